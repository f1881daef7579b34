"""CPU: refusals of the paged-cache and batch-sampling entry points (every one returns before a
launch), and the 64-bit forms that the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

import _paged as P
from jieyu_b200 import _capi

A = 1 << 20  # a pointer value that no refused call may follow


def _pages(**kw):
    d = dict(k=A, ks=A, v=A, vs=A, num_pages=4, page_size=16, page_stride=16 * 2 * 64, pos_stride=128, head_stride=64,
             spage_stride=32, spos_stride=2, shead_stride=1)
    d.update(kw)
    return _capi.KVPages(**d)


BAD_PAGES = [dict(k=None), dict(ks=None), dict(v=None), dict(vs=None), dict(num_pages=0), dict(page_size=0),
             dict(page_size=-1), dict(k=A + 2), dict(v=A + 1), dict(ks=A + 2), dict(pos_stride=130),
             dict(head_stride=-64), dict(spage_stride=-1), dict(page_size=1 << 30)]


def _append(read=False, **kw):
    d = dict(K=A, V=A, ld=128, rows=3, kv=2, hd=64, seq=A, pos=A, table=A, width=8, seqs=3, cos=None, sin=None,
             rope=0, pages=_pages())
    d.update(kw)
    lib = _capi.load()
    p = C.byref(d["pages"]) if d["pages"] is not None else None
    head = (d["K"], d["V"], d["ld"], d["rows"], d["kv"], d["hd"], d["seq"], d["pos"], d["table"], d["width"], d["seqs"])
    if read:
        return lib.jyc_kv_read_paged_q8(*head, p, None)
    return lib.jyc_kv_append_paged_q8(*head, d["cos"], d["sin"], d["rope"], p, None)


def _attend(**kw):
    d = dict(Q=A, ldq=256, out=A, ldo=256, H=4, kv=2, hd=64, lens=A, table=A, width=8, seqs=3, cos=None, sin=None,
             rope=0, pages=_pages(), work=None, bytes=0)
    d.update(kw)
    p = C.byref(d["pages"]) if d["pages"] is not None else None
    return _capi.load().jyc_attention_paged_q8(d["Q"], d["ldq"], d["out"], d["ldo"], d["H"], d["kv"], d["hd"],
                                               d["lens"], d["table"], d["width"], d["seqs"], d["cos"], d["sin"],
                                               d["rope"], p, d["work"], d["bytes"], None)


SHARED = [dict(kv=0), dict(kv=-2), dict(hd=0), dict(hd=62), dict(hd=260), dict(table=None), dict(width=-1),
          dict(seqs=-1), dict(cos=A), dict(sin=A), dict(cos=A, sin=A, rope=0), dict(pages=None)]


@pytest.mark.parametrize("kw", SHARED + [dict(rows=-1), dict(ld=127), dict(K=None), dict(V=None), dict(pos=None),
                                         dict(seq=None, rows=4)])
def test_append_and_read_refuse(kw):
    assert _append(**kw) == _capi.JYC_ERR_ARG
    assert "kv_append_paged_q8" in _capi.last_error()
    if not {"cos", "sin"} & set(kw):
        assert _append(read=True, **kw) == _capi.JYC_ERR_ARG
        assert "kv_read_paged_q8" in _capi.last_error()


@pytest.mark.parametrize("kw", BAD_PAGES)
def test_bad_pages_are_refused(kw):
    assert _append(pages=_pages(**kw)) == _capi.JYC_ERR_ARG
    assert _append(read=True, pages=_pages(**kw)) == _capi.JYC_ERR_ARG
    assert _attend(pages=_pages(**kw)) == _capi.JYC_ERR_ARG


@pytest.mark.parametrize("kw", SHARED + [dict(H=0), dict(H=3), dict(H=-2), dict(ldq=255), dict(ldo=255), dict(Q=None),
                                         dict(out=None), dict(lens=None)])
def test_attention_refuses(kw):
    assert _attend(**kw) == _capi.JYC_ERR_ARG
    assert "attention_paged_q8" in _capi.last_error()


def test_empty_calls_do_nothing():
    assert _append(rows=0, K=None, V=None, pos=None) == _capi.JYC_OK
    assert _append(read=True, rows=0, K=None, V=None, pos=None) == _capi.JYC_OK
    assert _attend(seqs=0, Q=None, out=None, lens=None) == _capi.JYC_OK
    assert _capi.load().jyc_sample_batch(None, 8, 0, 8, None, None, None, None, None, None, None, None) == _capi.JYC_OK


def test_workspace_query_refuses_bad_shapes():
    f = _capi.load().jyc_attention_paged_q8_workspace
    for bad in ((-1, 4, 2, 64), (1, 4, 3, 64), (1, 0, 2, 64), (1, 4, 0, 64), (1, 4, 2, 65), (1, 4, 2, 260)):
        assert f(*bad) == 0
        assert "workspace" in _capi.last_error()


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(V=0), dict(V=-3), dict(V=(1 << 20) + 1, ld=1 << 21), dict(ld=99),
                                dict(logits=None), dict(u=None), dict(ids=None)])
def test_sample_batch_refuses(kw):
    d = dict(logits=A, ld=100, rows=2, V=100, u=A, ids=A)
    d.update(kw)
    assert _capi.load().jyc_sample_batch(d["logits"], d["ld"], d["rows"], d["V"], None, None, None, None, d["u"],
                                         d["ids"], None, None) == _capi.JYC_ERR_ARG
    assert "sample_batch" in _capi.last_error()


def test_plain_rotation_and_rounding_equal_the_oracle(oracle):
    """The 64-bit forms reproduce rope_pos and kv_pack_q8 bit for bit."""
    rng = np.random.default_rng(5)
    for hd in (4, 36, 64, 80, 128, 256):
        n, heads, start = 9, 3, 11
        x = rng.normal(size=(n, heads, hd)).astype(np.float32)
        cos, sin = P.tables(start + n, hd)
        want = x.copy()
        oracle.rope_pos(want.ctypes.data, n, start, heads, hd, cos.ctypes.data, sin.ctypes.data)
        got = P.rotate(x.astype(np.float64), np.arange(start, start + n), cos, sin)
        assert np.array_equal(got.astype(np.float32), want), hd
        q8, sc = np.empty((n, heads, hd), np.int8), np.empty((n, heads), np.float32)
        want[2] = 0.0
        want[3] *= np.float32(1e-9)
        oracle.kv_pack_q8(want.ctypes.data, q8.ctypes.data, sc.ctypes.data, heads, hd, n)
        q, s = P.quantise(want.astype(np.float64))
        assert np.array_equal(q.astype(np.int8), q8) and np.array_equal(s.astype(np.float32), sc), hd


def test_plain_picks():
    l = np.array([0.0, 3.0, np.nan, 3.0, -np.inf, 1.0], np.float32)
    assert P.picks(l, 0.0, None, None, None, 0.5) == {1: 1.0}
    assert set(P.picks(l, 1.0, 1, None, None, 0.99)) == {1}
    assert set(P.picks(l, 1.0, 2, None, None, 0.6)) == {3}
    assert set(P.picks(l, 1.0, None, 0.3, None, 0.7)) == {1}
    assert set(P.picks(l, 1.0, None, None, 1.0, 0.75)) == {3}
    assert P.picks(np.full(4, -np.inf, np.float32), 1.0, None, None, None, 0.5) == {-1: 0.0}
