"""CPU: refusals of the rotary-row, 8-bit product and 4-bit cache entry points (every one returns
before a launch), and the scaled RoPE tables."""
import ctypes as C
import math

import numpy as np
import pytest

from jieyu_b200 import _capi
from jieyu_b200.model import rope_table

A = 1 << 20  # a pointer value that no refused call may follow


def _pages(**kw):
    d = dict(k=A, kp=A, v=A, vp=A, mass=A, num_pages=4, page_size=16, page_stride=16 * 2 * 32, pos_stride=64,
             head_stride=32, ppage_stride=64, ppos_stride=4, phead_stride=2, mpage_stride=32, mpos_stride=2,
             mhead_stride=1)
    d.update(kw)
    return _capi.KVPagesQ4(**d)


def _rope(**kw):
    d = dict(cos_table=A, sin_table=A, len=8, rot_dim=64, layout=_capi.JYC_ROPE_HALVES)
    d.update(kw)
    return _capi.Rope(**d)


def _ref(x):
    return None if x is None else C.byref(x)


def _append(read=False, **kw):
    d = dict(K=A, V=A, ld=128, rows=3, kv=2, hd=64, seq=A, pos=A, table=A, width=8, seqs=3, rope=None, rope_pos=None,
             pages=_pages())
    d.update(kw)
    lib = _capi.load()
    head = (d["K"], d["V"], d["ld"], d["rows"], d["kv"], d["hd"], d["seq"], d["pos"], d["table"], d["width"], d["seqs"])
    if read:
        return lib.jyc_kv_read_paged_q4(*head, _ref(d["pages"]), None)
    return lib.jyc_kv_append_paged_q4(*head, _ref(d["rope"]), d["rope_pos"], _ref(d["pages"]), None)


def _attend(**kw):
    d = dict(Q=A, ldq=256, out=A, ldo=256, H=4, kv=2, hd=64, lens=A, table=A, width=8, seqs=3, rope=None,
             rope_pos=None, pages=_pages(), work=None, bytes=0)
    d.update(kw)
    return _capi.load().jyc_attention_paged_q4(d["Q"], d["ldq"], d["out"], d["ldo"], d["H"], d["kv"], d["hd"],
                                               d["lens"], d["table"], d["width"], d["seqs"], _ref(d["rope"]),
                                               d["rope_pos"], _ref(d["pages"]), d["work"], d["bytes"], None)


def _evict(**kw):
    d = dict(lens=A, budget=32, recent=8, kv=2, hd=64, table=A, width=8, seqs=3, new=A, new_width=2, new_lens=2 * A,
             kept=A, pages=_pages())
    d.update(kw)
    return _capi.load().jyc_kv_evict_paged_q4(d["lens"], d["budget"], d["recent"], d["kv"], d["hd"], d["table"],
                                              d["width"], d["seqs"], d["new"], d["new_width"], d["new_lens"],
                                              d["kept"], _ref(d["pages"]), None)


SHARED = [dict(kv=0), dict(kv=-2), dict(hd=0), dict(hd=62), dict(hd=260), dict(table=None), dict(width=-1),
          dict(seqs=-1), dict(pages=None)]
BAD_PAGES = [dict(k=None), dict(kp=None), dict(v=None), dict(vp=None), dict(num_pages=0), dict(page_size=0),
             dict(page_size=-1), dict(k=A + 8), dict(v=A + 4), dict(kp=A + 2), dict(vp=A + 1), dict(mass=A + 2),
             dict(pos_stride=72), dict(head_stride=-32), dict(ppage_stride=-1), dict(mhead_stride=-1),
             dict(page_size=1 << 30)]
BAD_ROPES = [dict(cos_table=None), dict(sin_table=None), dict(cos_table=A + 2), dict(len=0), dict(rot_dim=0),
             dict(rot_dim=63), dict(rot_dim=66), dict(layout=2), dict(layout=-1)]


@pytest.mark.parametrize("kw", SHARED + [dict(rows=-1), dict(ld=127), dict(K=None), dict(V=None), dict(pos=None),
                                         dict(seq=None, rows=4)])
def test_append_and_read_refuse(kw):
    assert _append(**kw) == _capi.JYC_ERR_ARG
    assert "kv_append_paged_q4" in _capi.last_error()
    assert _append(read=True, **kw) == _capi.JYC_ERR_ARG
    assert "kv_read_paged_q4" in _capi.last_error()


@pytest.mark.parametrize("kw", BAD_PAGES)
def test_bad_pages_are_refused(kw):
    p = _pages(**kw)
    for call in (_append, _attend, _evict, lambda **k: _append(read=True, **k)):
        assert call(pages=p) == _capi.JYC_ERR_ARG


@pytest.mark.parametrize("kw", BAD_ROPES)
def test_bad_ropes_are_refused(kw):
    r = _rope(**kw)
    assert _append(rope=r) == _capi.JYC_ERR_ARG
    assert _attend(rope=r) == _capi.JYC_ERR_ARG
    assert _turn(rope=r) == _capi.JYC_ERR_ARG


@pytest.mark.parametrize("kw", SHARED + [dict(H=0), dict(H=3), dict(H=-2), dict(ldq=255), dict(ldo=255), dict(Q=None),
                                         dict(out=None), dict(lens=None), dict(seqs=1 << 30)])
def test_attention_refuses(kw):
    assert _attend(**kw) == _capi.JYC_ERR_ARG
    assert "attention_paged_q4" in _capi.last_error()


@pytest.mark.parametrize("kw", SHARED + [dict(budget=0), dict(budget=-1), dict(recent=-1), dict(recent=33),
                                         dict(new_width=1), dict(new_width=-1), dict(lens=None), dict(new=None),
                                         dict(new_lens=None), dict(kept=None), dict(new_lens=A), dict(seqs=1 << 26),
                                         dict(pages=_pages(mass=None))])
def test_eviction_refuses(kw):
    assert _evict(**kw) == _capi.JYC_ERR_ARG
    assert "kv_evict_paged_q4" in _capi.last_error()


def test_workspace_query_refuses_bad_shapes():
    f = _capi.load().jyc_attention_paged_q4_workspace
    for bad in ((-1, 4, 2, 64, 0), (1, 4, 3, 64, 0), (1, 0, 2, 64, 0), (1, 4, 0, 64, 0), (1, 4, 2, 65, 0),
                (1, 4, 2, 260, 0), (1, 4, 2, 64, -1), (1, 4, 2, 64, 0x7fffff01), (1 << 30, 4, 2, 64, 0)):
        assert f(*bad) == 0
        assert "workspace" in _capi.last_error()


def test_more_scores_than_bytes_count_are_refused():
    """A workspace of 2^64 bytes and more: its size would come out small, and the scores would lie behind it."""
    f = _capi.load().jyc_attention_paged_q4_workspace
    for H, kv in ((16, 16), (16, 1), (15, 3)):
        assert f(1 << 27, H, kv, 4, 0x7fffff00) == 0
        assert "bad shape" in _capi.last_error()
        assert _attend(seqs=1 << 27, H=H, kv=kv, hd=4, width=1, pages=_pages(page_size=0x7fffff00)) == _capi.JYC_ERR_ARG
        assert "attention_paged_q4" in _capi.last_error()
    assert _attend(seqs=1 << 26, H=16, kv=16, hd=4, width=1, work=A, bytes=1 << 62,
                   pages=_pages(page_size=0x7fffff00)) == _capi.JYC_ERR_ARG


def _turn(**kw):
    d = dict(X=A, ldx=128, Y=2 * A, ldy=128, rows=3, heads=2, hd=64, pos=A, rope=_rope())
    d.update(kw)
    return _capi.load().jyc_rope_rows(d["X"], d["ldx"], d["Y"], d["ldy"], d["rows"], d["heads"], d["hd"], d["pos"],
                                      _ref(d["rope"]), None)


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(heads=0), dict(hd=0), dict(ldx=127), dict(ldy=127), dict(X=None),
                                dict(Y=None), dict(pos=None), dict(rope=None), dict(Y=A, ldy=130)])
def test_rope_rows_refuses(kw):
    assert _turn(**kw) == _capi.JYC_ERR_ARG
    assert "rope_rows" in _capi.last_error()


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(k=0), dict(ldx=99), dict(ldq=99), dict(x=None), dict(q=None),
                                dict(scale=None)])
def test_quantize_rows_refuses(kw):
    d = dict(x=A, ldx=100, rows=2, k=100, q=A, ldq=100, scale=A)
    d.update(kw)
    assert _capi.load().jyc_quantize_rows_i8(*d.values(), None) == _capi.JYC_ERR_ARG
    assert "quantize_rows_i8" in _capi.last_error()


@pytest.mark.parametrize("kw", [dict(m=-1), dict(n=0), dict(k=0), dict(k=131072, lda=131072, ldw=131072),
                                dict(lda=96), dict(ldw=96), dict(lda=113), dict(ldw=120), dict(ldc=39), dict(A=None),
                                dict(a_scale=None), dict(W=None), dict(w_scale=None), dict(C=None), dict(A=A + 8),
                                dict(W=A + 4)])
def test_matmul_i8_refuses(kw):
    d = dict(A=A, lda=112, a_scale=A, W=A, ldw=112, w_scale=A, bias=None, C=A, ldc=40, m=3, n=40, k=100)
    d.update(kw)
    assert _capi.load().jyc_matmul_i8(*d.values(), None) == _capi.JYC_ERR_ARG
    assert "matmul_i8" in _capi.last_error()


@pytest.mark.parametrize("kw", [dict(m=2**31 - 255), dict(m=2**31 - 1), dict(n=2**31 - 255, ldc=2**31 - 1),
                                dict(n=2**31 - 1, ldc=2**31 - 1)])
def test_matmul_i8_refuses_more_tiles_than_an_int_counts(kw):
    """A tile of 256 channels or tokens that starts below 2^31 must also end there: places are counted in ints."""
    d = dict(A=A, lda=16, a_scale=A, W=A, ldw=16, w_scale=A, bias=None, C=A, ldc=40, m=3, n=40, k=16)
    d.update(kw)
    assert _capi.load().jyc_matmul_i8(*d.values(), None) == _capi.JYC_ERR_ARG
    assert "matmul_i8" in _capi.last_error()


@pytest.mark.parametrize("k", [2**31 - 1023, 2**31 - 1])
def test_quantize_rows_refuses_rows_that_an_int_steps_over(k):
    """256 threads take quads of a row in turn: the step behind the last one must stay below 2^31."""
    assert _capi.load().jyc_quantize_rows_i8(A, 2**31 - 1, 2, k, A, 2**31 - 1, A, None) == _capi.JYC_ERR_ARG
    assert "quantize_rows_i8" in _capi.last_error()


def test_empty_calls_do_nothing():
    lib = _capi.load()
    assert _append(rows=0, K=None, V=None, pos=None) == _capi.JYC_OK
    assert _append(read=True, rows=0, K=None, V=None, pos=None) == _capi.JYC_OK
    assert _attend(seqs=0, Q=None, out=None, lens=None) == _capi.JYC_OK
    assert _evict(seqs=0, lens=None, new=None, new_lens=None, kept=None) == _capi.JYC_OK
    assert _turn(rows=0, X=None, Y=None, pos=None) == _capi.JYC_OK
    assert lib.jyc_quantize_rows_i8(None, 8, 0, 8, None, 8, None, None) == _capi.JYC_OK
    assert lib.jyc_matmul_i8(None, 16, None, None, 16, None, None, None, 8, 0, 8, 16, None) == _capi.JYC_OK


# ---- scaled tables -----------------------------------------------------------


def _table(n, r, theta, scaling):
    c, s = np.full((n, r // 2), 9.0, np.float32), np.full((n, r // 2), 9.0, np.float32)
    _capi.check(_capi.load().jyc_rope_table_scaled(n, r, theta, _ref(scaling), c.ctypes.data, s.ctypes.data))
    return c, s


def _frequencies(r, theta, kind, factor, L, low, high):
    j = np.arange(r // 2)
    f = theta ** (-2.0 * j / r)
    if kind == _capi.JYC_ROPE_LINEAR:
        return f / factor
    if kind == _capi.JYC_ROPE_NTK:
        return (theta * factor ** (r / (r - 2.0))) ** (-2.0 * j / r)
    if kind == _capi.JYC_ROPE_BANDS:
        t = np.clip((L * f / (2 * math.pi) - low) / (high - low), 0, 1)
        return f * ((1 - t) / factor + t)
    if kind == _capi.JYC_ROPE_RAMP:
        at = lambda turns: r * math.log(L / (2 * math.pi * turns)) / (2 * math.log(theta))  # noqa: E731
        a, b = max(math.floor(at(high)), 0), min(math.ceil(at(low)), r - 1)
        t = 1 - np.clip((j - a) / (b - a), 0, 1)
        return f * ((1 - t) / factor + t)
    return f


@pytest.mark.parametrize("kind,factor,L,low,high,attention", [
    (_capi.JYC_ROPE_NONE, 1.0, 0, 0.0, 0.0, 0.0), (_capi.JYC_ROPE_LINEAR, 4.0, 0, 0.0, 0.0, 0.0),
    (_capi.JYC_ROPE_NTK, 8.0, 0, 0.0, 0.0, 0.0), (_capi.JYC_ROPE_BANDS, 8.0, 8192, 1.0, 4.0, 0.0),
    (_capi.JYC_ROPE_RAMP, 16.0, 4096, 1.0, 32.0, 0.0), (_capi.JYC_ROPE_RAMP, 40.0, 4096, 1.0, 32.0, 1.5)])
@pytest.mark.parametrize("r,theta", [(64, 1e4), (128, 5e5), (20, 1e4)])
def test_scaled_tables(kind, factor, L, low, high, attention, r, theta):
    n = 700
    c, s = _table(n, r, theta, _capi.RopeScaling(kind, factor, L, low, high, attention))
    gain = (attention or 0.1 * math.log(factor) + 1) if kind == _capi.JYC_ROPE_RAMP else 1.0
    angle = np.arange(n)[:, None] * _frequencies(r, theta, kind, factor, L, low, high)
    # one rounding of a number up to gain, and 1e-12 for an angle below 700 in 64 bits (the 32-bit constants aside,
    # which both sides take as they are)
    tol = gain * (2.0 ** -24 + 1e-12)
    assert np.abs(c - gain * np.cos(angle)).max() <= tol and np.abs(s - gain * np.sin(angle)).max() <= tol


def test_unscaled_table_is_near_the_reference_table():
    c, s = _table(100, 64, 1e4, None)
    rc, rs = rope_table(100, 64, 1e4)
    # the reference's frequency and angle are rounded to 32 bits: an angle below 100 is off by at most 100 * 4 half
    # steps (powf's error included), its cosine by as much and two more roundings
    assert np.abs(c - rc.reshape(c.shape)).max() <= 100 * 6 * 2.0 ** -24
    assert np.abs(s - rs.reshape(s.shape)).max() <= 100 * 6 * 2.0 ** -24


@pytest.mark.parametrize("args,scaling", [
    ((0, 64, 1e4), None), ((8, 63, 1e4), None), ((8, 0, 1e4), None), ((8, 64, 0.0), None), ((8, 64, math.nan), None),
    ((8, 64, 1e4), _capi.RopeScaling(5, 2.0, 0, 0, 0, 0)), ((8, 64, 1e4), _capi.RopeScaling(-1, 2.0, 0, 0, 0, 0)),
    ((8, 64, 1e4), _capi.RopeScaling(1, 0.5, 0, 0, 0, 0)), ((8, 64, 1e4), _capi.RopeScaling(1, math.nan, 0, 0, 0, 0)),
    ((8, 2, 1e4), _capi.RopeScaling(2, 2.0, 0, 0, 0, 0)), ((8, 64, 1e4), _capi.RopeScaling(3, 2.0, 0, 1, 4, 0)),
    ((8, 64, 1e4), _capi.RopeScaling(3, 2.0, 8, 4, 4, 0)), ((8, 64, 1e4), _capi.RopeScaling(4, 2.0, 8, 0, 4, 0)),
    ((8, 64, 1.0), _capi.RopeScaling(4, 2.0, 8, 1, 4, 0)), ((8, 64, 1e4), _capi.RopeScaling(4, 2.0, 8, 1, 4, -1))])
def test_scaled_tables_refuse(args, scaling):
    buf = np.zeros(8 * 32, np.float32)
    assert _capi.load().jyc_rope_table_scaled(*args, _ref(scaling), buf.ctypes.data, buf.ctypes.data) == _capi.JYC_ERR_ARG
    assert "rope_table_scaled" in _capi.last_error()


@pytest.mark.parametrize("call,names", [
    (_append, ("K", "V", "seq", "pos", "rope_pos")), (lambda **k: _append(read=True, **k), ("K", "V", "seq", "pos")),
    (_attend, ("Q", "out", "lens", "rope_pos")), (_evict, ("lens", "new", "new_lens", "kept")), (_turn, ("X", "Y", "pos"))])
def test_misaligned_arrays_are_refused(call, names):
    for name in names:
        assert call(**{name: 4 * A + 2}) == _capi.JYC_ERR_ARG
        assert "misaligned" in _capi.last_error()


@pytest.mark.parametrize("name", ["a_scale", "w_scale", "bias", "C"])
def test_misaligned_scales_are_refused(name):
    d = dict(A=A, lda=112, a_scale=A, W=A, ldw=112, w_scale=A, bias=None, C=A, ldc=40, m=3, n=40, k=100)
    d[name] = A + 1
    assert _capi.load().jyc_matmul_i8(*d.values(), None) == _capi.JYC_ERR_ARG
    assert "misaligned" in _capi.last_error()
    assert _capi.load().jyc_quantize_rows_i8(A + 2, 100, 2, 100, A, 100, A, None) == _capi.JYC_ERR_ARG
