"""The paged int8 cache on the device (jyc_kv_append_paged_q8, jyc_kv_read_paged_q8,
jyc_attention_paged_q8) against the plain 64-bit forms of _paged.py.

Bytes, scales and read-back values are equal bit for bit (each is a defined fp32 rounding);
attention is within the rounding bound that _paged.attention_tolerance derives.
"""
import ctypes as C

import numpy as np
import pytest

import _paged as P
from _util import dev, host
from jieyu_b200 import _capi

pytestmark = pytest.mark.gpu


def _stream(torch):
    return torch.cuda.current_stream().cuda_stream


def _append(torch, pool, K, V, ld, rows, seq, pos, cos=None, sin=None):
    return _capi.load().jyc_kv_append_paged_q8(
        K, V, ld, rows, pool.kv, pool.hd, P.ptr(seq), P.ptr(pos), P.ptr(pool.table), pool.table.shape[1],
        pool.table.shape[0], P.ptr(cos), P.ptr(sin), 0 if cos is None else cos.shape[0], C.byref(pool.desc),
        _stream(torch))


def _read(torch, pool, K, V, ld, rows, seq, pos):
    return _capi.load().jyc_kv_read_paged_q8(
        K, V, ld, rows, pool.kv, pool.hd, P.ptr(seq), P.ptr(pos), P.ptr(pool.table), pool.table.shape[1],
        pool.table.shape[0], C.byref(pool.desc), _stream(torch))


def _table(rng, seqs, width, spare=3):
    pages = seqs * width + spare
    return pages, rng.permutation(pages)[: seqs * width].reshape(seqs, width)


@pytest.fixture(autouse=True)
def no_error_left(cuda):
    lib = _capi.load()
    lib.jyc_paged_error(1)
    yield
    assert lib.jyc_paged_error(1) == 0


# ---- append and read ---------------------------------------------------------

APPEND = [  # kv, hd, page, heads_first, rope, ld beyond the heads, gap behind each row, offset of K in floats
    (2, 64, 16, False, True, 0, 0, 0),
    (8, 128, 32, True, True, 8, 0, 0),
    (3, 80, 7, False, True, 3, 4, 0),      # rows not 16-byte aligned
    (1, 4, 1, True, True, 0, 0, 1),        # smallest head, one position a page, misaligned input
    (5, 36, 257, False, False, 0, 12, 2),
    (2, 256, 16, True, True, 4, 0, 0),
    (4, 132, 5, False, False, 0, 0, 0),
    (16, 96, 64, True, False, 0, 32, 4),
]


@pytest.mark.parametrize("kv,hd,page,hf,rope,extra,gap,off", APPEND)
@pytest.mark.parametrize("rows", [1, 37, 300])
def test_append_and_read_back(cuda, kv, hd, page, hf, rope, extra, gap, off, rows):
    torch = cuda
    rng = np.random.default_rng(rows * 1000 + hd)
    seqs = min(rows, 5)
    width = (rows + 9) // page + 1
    pages, table = _table(rng, seqs, width)
    pool = P.Pool(torch, pages, page, kv, hd, table, hf, gap, fill=77)
    seq = np.arange(rows) % seqs
    pos = np.arange(rows) // seqs + rng.integers(0, 5)
    pad = rng.random(rows) < 0.2
    pos[pad] = -1 - rng.integers(0, 5, pad.sum())
    ld = 2 * kv * hd + extra
    x = rng.normal(size=rows * ld + off).astype(np.float32)
    if rows > 4:
        r = x[off:].reshape(rows, ld)
        r[1, :hd] = 0.0                        # scale 0
        r[2, :hd] = 1e-9                       # below the threshold
        r[3, hd // 2] = 3e38
        r[4, :hd] *= np.float32(1e-30)
    xd, seqd, posd = dev(torch, x), dev(torch, seq.astype(np.int32)), dev(torch, pos.astype(np.int32))
    cos = sin = None
    if rope:
        c, s = P.tables(width * page, hd)
        cos, sin = dev(torch, c), dev(torch, s)
    base = xd.data_ptr() + 4 * off
    before = [t.clone() for t in (pool.k8, pool.v8, pool.ks, pool.vs)]
    _capi.check(_append(torch, pool, base, base + 4 * kv * hd, ld, rows, seqd, posd, cos, sin))
    body = x[off:].reshape(rows, ld).astype(np.float64)
    Kh = body[:, : kv * hd].reshape(rows, kv, hd)
    Vh = body[:, kv * hd: 2 * kv * hd].reshape(rows, kv, hd)
    if rope:
        Kh = P.rotate(Kh, np.maximum(pos, 0), c, s)
    (kq, ks), (vq, vs) = P.quantise(Kh), P.quantise(Vh)
    # the whole pool: named slots hold the rows, everything else is as it was
    k8, v8, kss, vss = (host(t) for t in (pool.k8, pool.v8, pool.ks, pool.vs))
    wk, wv, wks, wvs = (host(t).copy() for t in before)
    for i in range(rows):
        if pos[i] < 0:
            continue
        pg, sl = table[seq[i], pos[i] // page], pos[i] % page
        idx = (pg, slice(None), sl) if hf else (pg, sl)
        wk[idx][:, :hd], wv[idx][:, :hd] = kq[i].astype(np.int8), vq[i].astype(np.int8)
        wks[idx], wvs[idx] = ks[i].astype(np.float32), vs[i].astype(np.float32)
    assert np.array_equal(k8, wk) and np.array_equal(v8, wv)
    assert np.array_equal(kss, wks, equal_nan=True) and np.array_equal(vss, wvs, equal_nan=True)
    # read back: q * scale in fp32; rows without a position and columns behind the heads stay
    back = torch.full((rows * ld + off,), -7.0, device="cuda")
    bb = back.data_ptr() + 4 * off
    _capi.check(_read(torch, pool, bb, bb + 4 * kv * hd, ld, rows, seqd, posd))
    got = host(back)
    want = np.full((rows, ld), -7.0, np.float32)
    live = pos >= 0
    want[live, : kv * hd] = (kq * ks[..., None])[live].reshape(-1, kv * hd).astype(np.float32)
    want[live, kv * hd: 2 * kv * hd] = (vq * vs[..., None])[live].reshape(-1, kv * hd).astype(np.float32)
    assert np.all(got[:off] == -7.0)
    assert np.array_equal(got[off:].reshape(rows, ld), want)


def test_append_equals_kv_pack_q8(cuda):
    """Without RoPE the bytes and scales are jyc_kv_pack_q8's; infinities and NaN among the values too."""
    torch = cuda
    rng = np.random.default_rng(3)
    kv, hd, n = 4, 64, 12
    x = rng.normal(size=(n, kv, hd)).astype(np.float32)
    x[1, 0, 3] = np.inf
    x[2, 1, 5] = np.nan
    x[3, 2] = -np.inf
    x[4, 3] = np.nan
    xd = dev(torch, x)
    q = torch.empty(n * kv * hd, dtype=torch.int8, device="cuda")
    s = torch.empty(n * kv, device="cuda")
    _capi.check(_capi.load().jyc_kv_pack_q8(xd.data_ptr(), q.data_ptr(), s.data_ptr(), kv, hd, n, _stream(torch)))
    pool = P.Pool(torch, 1, n, kv, hd, [[0]])
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    seq = torch.zeros_like(pos)
    _capi.check(_append(torch, pool, xd.data_ptr(), xd.data_ptr(), kv * hd, n, seq, pos))
    for t8, ts in ((pool.k8, pool.ks), (pool.v8, pool.vs)):
        assert np.array_equal(host(t8).ravel(), host(q))
        assert np.array_equal(host(ts).ravel(), host(s), equal_nan=True)


def test_out_of_range_rows_are_skipped_and_flagged(cuda):
    torch = cuda
    lib = _capi.load()
    kv, hd, page = 2, 64, 4
    table = np.array([[0, 1], [2, 99], [-3, 3]], np.int32)
    rng = np.random.default_rng(0)
    x = dev(torch, rng.normal(size=(1, 2 * kv * hd)).astype(np.float32))
    c, s = P.tables(6, hd)
    cos, sin = dev(torch, c), dev(torch, s)
    for seq, pos, rope, bit in ((3, 0, False, 1), (-1, 0, False, 1), (0, 8, False, 1), (0, 2 ** 31 - 1, False, 1),
                                (1, 4, False, 2), (2, 1, False, 2), (0, 6, True, 4)):
        pool = P.Pool(torch, 4, page, kv, hd, table, fill=55)
        seqd = torch.tensor([seq], dtype=torch.int32, device="cuda")
        posd = torch.tensor([pos], dtype=torch.int32, device="cuda")
        _capi.check(_append(torch, pool, x.data_ptr(), x.data_ptr(), kv * hd, 1, seqd, posd, cos if rope else None,
                            sin if rope else None))
        assert lib.jyc_paged_error(1) == bit, (seq, pos)
        assert lib.jyc_paged_error(0) == 0
        assert bool((pool.k8 == 55).all()) and bool((pool.v8 == 55).all()) and bool(pool.ks.isnan().all())
        if not rope:
            back = torch.full((2, kv * hd), 3.0, device="cuda")
            _capi.check(_read(torch, pool, back.data_ptr(), back.data_ptr() + 4 * kv * hd, kv * hd, 1, seqd, posd))
            assert lib.jyc_paged_error(1) == bit
            assert bool((back == 3.0).all())


# ---- attention ---------------------------------------------------------------

def _check(torch, pool, q, lens, H, out, rope=None, rows=None):
    """Every row of `out` against the 64-bit form on the pool's own bytes."""
    hd = pool.hd
    for b in (range(len(lens)) if rows is None else rows):
        n = int(lens[b])
        got = out[b, : H * hd].reshape(H, hd)
        if n <= 0:
            assert np.all(got == 0.0), b
            continue
        x = q[b, : H * hd].astype(np.float64).reshape(1, H, hd)
        if rope is not None:
            x = P.rotate(x, np.array([n - 1]), *rope)
        qq, qs = P.quantise(x[0])
        k, ks, v, vs = pool.rows(b, n)
        want = P.attention(qq, qs, k, ks, v, vs)
        g = H // pool.kv
        smax = max(np.abs((k[:, h // g] @ qq[h]) * ks[:, h // g] * qs[h]).max() for h in range(H)) / np.sqrt(hd)
        vmax = np.abs(v * vs[..., None]).max()
        err = np.abs(got - want).max()
        assert err <= P.attention_tolerance(n, smax, vmax), (b, n, err, P.attention_tolerance(n, smax, vmax))


ATTEND = [  # H, KV, hd, page, heads_first, rope, gap, lengths
    (14, 2, 64, 16, False, True, 0, [513, 1, 0, 16, 17, 15]),
    (32, 8, 64, 32, True, True, 0, [2100, 31, 32, 33, 64, 65, 0, 1]),
    (32, 8, 128, 64, False, False, 0, [700, 4096, 3]),
    (4, 4, 128, 1, False, True, 0, [1, 2, 63, 100]),          # one query head a kv head, one position a page
    (2, 1, 256, 257, True, True, 0, [257, 258, 900]),
    (9, 1, 96, 7, False, True, 16, [50, 0, 333]),              # more than 8 query heads a kv head
    (32, 2, 80, 13, True, False, 0, [29, 500]),
    (24, 1, 192, 16, False, True, 0, [100, 1]),                # more than 16
    (40, 2, 64, 5, True, True, 16, [77, 1025]),
    (7, 1, 36, 16, False, True, 0, [40, 129]),                 # rows not 16-byte aligned
    (3, 3, 4, 8, True, True, 0, [9, 100]),                     # smallest head
    (8, 2, 132, 16, False, False, 0, [70]),
    (2, 2, 252, 16, False, True, 4, [70, 300]),
    (6, 2, 64, 16, False, False, 4, [70, 300]),                # 16-byte heads at 4-byte strides
    (8, 2, 64, 1, False, True, 0, [5, 100]),                   # pages of 1, 2, 4, 8 and 96 positions
    (8, 2, 64, 2, True, True, 0, [5, 100]),
    (12, 1, 128, 1, True, True, 0, [33, 95]),
    (4, 2, 128, 4, False, False, 16, [33, 95]),
    (16, 2, 128, 8, True, True, 0, [260, 31]),
    (20, 2, 64, 96, False, True, 0, [96, 97, 500]),
    (8, 1, 128, 2048, False, True, 0, [2049, 100]),    (14, 2, 192, 16, True, True, 0, [300, 33]),                # large heads, 5 to 8 of them and more
    (16, 2, 256, 32, False, True, 0, [300, 17]),
    (22, 2, 256, 16, True, False, 0, [130, 1000]),
]


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "%dx%dx%d_p%d" % c[:4])
@pytest.mark.parametrize("own_work", [True, False])
def test_attention(cuda, case, own_work):
    torch = cuda
    H, KV, hd, page, hf, rope, gap, lens = case
    rng = np.random.default_rng(H * hd + page)
    width = max(lens) // page + 1
    pages, table = _table(rng, len(lens), width)
    # never-written places hold NaN scales: they must not reach a result
    pool = P.Pool(torch, pages, page, KV, hd, table, hf, gap, fill=-128)
    for b, n in enumerate(lens):
        pool.put_random(rng, b, n)
    ldq, ldo, B = H * hd + 5, H * hd + 3, len(lens)
    q = (2 * rng.normal(size=(B, ldq))).astype(np.float32)
    q[0, :hd] = 0.0                            # a query of zeros: equal weights
    tabs = P.tables(max(lens), hd) if rope else None
    qd = dev(torch, q)
    cos, sin = (dev(torch, t) for t in tabs) if rope else (None, None)
    out = torch.full((B + 1, ldo), -5.0, device="cuda")
    lensd = dev(torch, np.array(lens, np.int32))
    work = P.workspace(torch, B, H, KV, hd) if own_work else None
    _capi.check(P.attend(torch, pool, qd, out, H, lensd, cos, sin, work))
    got = host(out)
    assert np.all(got[B] == -5.0) and np.all(got[:, H * hd:] == -5.0)
    _check(torch, pool, q, lens, H, got, tabs)
    first = out.clone()
    _capi.check(P.attend(torch, pool, qd, out, H, lensd, cos, sin, work))
    assert np.array_equal(host(out), host(first))  # no order of execution in the result


@pytest.mark.parametrize("B,longest", [(300, 40), (1000, 3), (70, 900), (2, 20000)])
def test_attention_many_and_long(cuda, B, longest):
    torch = cuda
    H, KV, hd, page = 8, 2, 64, 16
    rng = np.random.default_rng(B)
    width = longest // page + 1
    lens = rng.integers(0, longest + 1, B)
    lens[0], lens[-1] = longest, 0
    # sequences share pages: the table repeats a pool of random ones
    pages = 4 * width
    table = rng.integers(0, pages, (B, width))
    table[0] = rng.permutation(pages)[:width]
    pool = P.Pool(torch, pages, page, KV, hd, table)
    pool2 = P.Pool(torch, pages, page, KV, hd, np.arange(pages)[None])
    pool2.k8, pool2.v8, pool2.ks, pool2.vs = pool.k8, pool.v8, pool.ks, pool.vs
    pool2.put_random(rng, 0, pages * page)
    q = rng.normal(size=(B, H * hd)).astype(np.float32)
    out = torch.empty(B, H * hd, device="cuda")
    _capi.check(P.attend(torch, pool, dev(torch, q), out, H, dev(torch, lens.astype(np.int32)),
                         work=P.workspace(torch, B, H, KV, hd)))
    rows = sorted(set(list(range(min(B, 12))) + list(range(B - 3, B)) + list(rng.integers(0, B, 20))))
    _check(torch, pool, q, lens, H, host(out), rows=rows)


def test_attention_sums_of_very_long_runs(cuda):
    """Runs of more than 2000 units of 32 keys with the largest digits there are: equal scores, every
    V byte 127. 1300 sequences of 131072 positions share one set of pages."""
    torch = cuda
    H, KV, hd, page, n, B = 2, 1, 64, 64, 131072, 1300
    pool = P.Pool(torch, n // page, page, KV, hd, np.tile(np.arange(n // page), (B, 1)))
    pool.v8.fill_(127)
    pool.ks.fill_(0.01)
    pool.vs.fill_(0.015)  # just below 2^-6: its weights have the largest fractions
    pool.k8.fill_(3)
    q = torch.randn(B, H * hd, device="cuda")
    out = torch.empty(B, H * hd, device="cuda")
    lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
    _capi.check(P.attend(torch, pool, q, out, H, lens, work=P.workspace(torch, B, H, KV, hd)))
    want = 127 * float(np.float32(0.015))
    # equal weights: the quotient of two sums, each of n / 32 rounded partial sums at most
    assert np.abs(host(out) - want).max() <= want * P.U24 * (2 * n / 32 + 64)


def test_attention_scales_that_are_not_finite(cuda):
    """A NaN or infinite scale of a key in range makes its heads' rows NaN, and no other row."""
    torch = cuda
    H, KV, hd, page = 8, 2, 64, 16
    rng = np.random.default_rng(3)
    for name, value in (("ks", np.nan), ("vs", np.nan), ("vs", np.inf)):
        pool = P.Pool(torch, 6, page, KV, hd, np.arange(6).reshape(2, 3))
        for b in range(2):
            pool.put_random(rng, b, 48)
        getattr(pool, "ks" if name == "ks" else "vs")[1, 5, 0] = value  # sequence 0, position 21, kv head 0
        q = rng.normal(size=(2, H * hd)).astype(np.float32)
        out = torch.empty(2, H * hd, device="cuda")
        lens = dev(torch, np.array([40, 48], np.int32))
        _capi.check(P.attend(torch, pool, dev(torch, q), out, H, lens, work=P.workspace(torch, 2, H, KV, hd)))
        got = host(out).reshape(2, H, hd)
        assert np.isnan(got[0, :4]).all() and np.isfinite(got[0, 4:]).all() and np.isfinite(got[1]).all()


@pytest.mark.parametrize("H,hd,side", [(4, 64, -1), (8, 128, 1), (16, 96, -1)])
def test_attention_infinite_key_scale(cuda, H, hd, side):
    """An infinite scale of K is not a weight of zero, whatever the sign of the key's dots."""
    torch = cuda
    page = 16
    rng = np.random.default_rng(5)
    pool = P.Pool(torch, 3, page, 1, hd, np.arange(3)[None])
    pool.put_random(rng, 0, 48)
    pool.k8[1, 5, 0, :] = side * 100
    pool.ks[1, 5, 0] = np.inf
    q = np.abs(rng.normal(size=(1, H * hd))).astype(np.float32)  # the dots with that key: all of its sign
    out = torch.empty(1, H * hd, device="cuda")
    lens = dev(torch, np.array([40], np.int32))
    _capi.check(P.attend(torch, pool, dev(torch, q), out, H, lens, work=P.workspace(torch, 1, H, 1, hd)))
    assert np.isnan(host(out)).all()


def test_attention_wide_range_of_scales(cuda):
    """V scales over 12 decades: the key with all the weight has the smallest one."""
    torch = cuda
    H, KV, hd, page, n = 8, 1, 64, 16, 200
    rng = np.random.default_rng(8)
    pool = P.Pool(torch, 13, page, KV, hd, rng.permutation(13)[None])
    pool.put_random(rng, 0, n)
    pool.ks.fill_(0.05)
    pool.vs.copy_(torch.from_numpy((10.0 ** rng.uniform(-10, 2, pool.vs.shape)).astype(np.float32)))
    pool.vs[int(pool.table_host[0, 3]), 2, 0] = 0.0
    q = (4 * rng.normal(size=(1, H * hd))).astype(np.float32)
    out = torch.empty(1, H * hd, device="cuda")
    lens = dev(torch, np.array([n], np.int32))
    _capi.check(P.attend(torch, pool, dev(torch, q), out, H, lens, work=P.workspace(torch, 1, H, KV, hd)))
    got = host(out).reshape(H, hd)
    k, ks, v, vs = pool.rows(0, n)
    qq, qs = P.quantise(q.astype(np.float64).reshape(H, hd))
    want = P.attention(qq, qs, k, ks, v, vs)
    for h in range(H):
        s = (k[:, 0] @ qq[h]) * ks[:, 0] * qs[h] / 8.0
        p = np.exp(s - s.max())
        p /= p.sum()
        # relative to the largest weighted row, not to the largest row of the cache
        top = (p * vs[:, 0]).max() * 127
        tol = P.attention_tolerance(n, np.abs(s).max(), 1.0) * (p * vs[:, 0] * 127).sum() + n * 2.0 ** -22 * top
        assert np.abs(got[h] - want[h]).max() <= tol, h


def test_attention_scores_of_every_size(cuda):
    """Scores to +-20000 (one key takes all), equal scores, and a first key far above the rest."""
    torch = cuda
    H, KV, hd, page, n = 2, 1, 128, 16, 100
    rng = np.random.default_rng(9)
    pool = P.Pool(torch, 7, page, KV, hd, np.arange(7)[None])
    pool.put_random(rng, 0, n)
    for ks in (1e3, 1e-12, 0.0):
        pool.ks.fill_(ks)
        q = (100 * rng.normal(size=(1, H * hd))).astype(np.float32)
        out = torch.empty(1, H * hd, device="cuda")
        lens = dev(torch, np.array([n], np.int32))
        _capi.check(P.attend(torch, pool, dev(torch, q), out, H, lens, work=P.workspace(torch, 1, H, KV, hd)))
        got = host(out).reshape(H, hd)
        k, kk, v, vs = pool.rows(0, n)
        qq, qs = P.quantise(q.astype(np.float64).reshape(H, hd))
        if ks == 1e3:  # the largest score leads by far more than its rounding
            for h in range(H):
                s = np.sort(k[:, 0] @ qq[h])
                assert (s[-1] - s[-2]) * ks * qs[h] / np.sqrt(hd) > 100
        want = P.attention(qq, qs, k, kk, v, vs)
        smax = 1.0 if ks == 1e3 else 1e-3  # one weight of 1 whatever the scores round to
        assert np.abs(got - want).max() <= P.attention_tolerance(n, smax, np.abs(v * vs[..., None]).max())


def test_attention_flags_what_is_out_of_range(cuda):
    torch = cuda
    lib = _capi.load()
    H, KV, hd, page = 4, 2, 64, 8
    rng = np.random.default_rng(4)
    table = np.array([[0, 1, 2, 3], [4, 5, 6, 7], [8, 9, 10, 11]], np.int32)
    pool = P.Pool(torch, 12, page, KV, hd, table)
    for b in range(3):
        pool.put_random(rng, b, 32)
    q = rng.normal(size=(3, H * hd)).astype(np.float32)
    qd = dev(torch, q)
    out = torch.empty(3, H * hd, device="cuda")
    work = P.workspace(torch, 3, H, KV, hd)
    # a length above the table's: cut to 32
    lens = dev(torch, np.array([33, 2 ** 31 - 1, -4], np.int32))
    _capi.check(P.attend(torch, pool, qd, out, H, lens, work=work))
    assert lib.jyc_paged_error(1) == 1
    _check(torch, pool, q, [32, 32, 0], H, host(out))
    # bad ids: their keys weigh nothing, the others' softmax stands
    pool.table[0, 1], pool.table[1, :] = 12, -1
    lens = dev(torch, np.array([20, 30, 9], np.int32))
    _capi.check(P.attend(torch, pool, qd, out, H, lens, work=work))
    assert lib.jyc_paged_error(1) == 2
    got = host(out)
    assert np.all(got[1] == 0.0)
    _check(torch, pool, q, [20, 30, 9], H, got, rows=[2])
    k, ks, v, vs = pool.rows(0, 20)
    keep = np.r_[0:8, 16:20]
    qq, qs = P.quantise(q[0].astype(np.float64).reshape(H, hd))
    want = P.attention(qq, qs, k[keep], ks[keep], v[keep], vs[keep])
    assert np.abs(got[0].reshape(H, hd) - want).max() <= P.attention_tolerance(20, 10.0, np.abs(v * vs[..., None]).max())
    # a query position behind the tables
    pool.table.copy_(torch.from_numpy(table))
    c, s = P.tables(10, hd)
    _capi.check(P.attend(torch, pool, qd, out, H, dev(torch, np.array([10, 11, 5], np.int32)), dev(torch, c),
                         dev(torch, s), work))
    assert lib.jyc_paged_error(1) == 4
    got = host(out)
    assert np.all(got[1] == 0.0)
    _check(torch, pool, q, [10, 11, 5], H, got, (c, s), rows=[0, 2])


def test_attention_small_workspace_is_refused(cuda):
    torch = cuda
    pool = P.Pool(torch, 2, 8, 2, 64, [[0, 1]])
    q = torch.zeros(1, 256, device="cuda")
    out = torch.zeros_like(q)
    lens = torch.ones(1, dtype=torch.int32, device="cuda")
    work = P.workspace(torch, 1, 4, 2, 64)
    assert P.attend(torch, pool, q, out, 4, lens, work=work[:-1]) == _capi.JYC_ERR_ARG
    assert "workspace too small" in _capi.last_error()
    big = torch.zeros(work.numel() + 16, dtype=torch.uint8, device="cuda")
    assert P.attend(torch, pool, q, out, 4, lens, work=big[4:]) == _capi.JYC_ERR_ARG
    assert "aligned" in _capi.last_error()


def test_attention_captured_replays_for_new_lengths(cuda):
    torch = cuda
    H, KV, hd, page, B = 8, 2, 64, 16, 6
    rng = np.random.default_rng(12)
    pages, table = _table(rng, B, 30)
    pool = P.Pool(torch, pages, page, KV, hd, table)
    for b in range(B):
        pool.put_random(rng, b, 480)
    tabs = P.tables(480, hd)
    cos, sin = (dev(torch, t) for t in tabs)
    qd = torch.empty(B, H * hd, device="cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    outs = [torch.empty(B, H * hd, device="cuda") for _ in range(2)]
    works = [P.workspace(torch, B, H, KV, hd), None]
    graphs = []
    for out, work in zip(outs, works):  # given workspace, and scratch inside the graph
        g = torch.cuda.CUDAGraph()
        P.attend(torch, pool, qd, out, H, lens, cos, sin, work)
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            _capi.check(P.attend(torch, pool, qd, out, H, lens, cos, sin, work))
        graphs.append(g)
    for n in ([480, 1, 0, 77, 300, 16], [0] * 6, [1, 2, 3, 4, 5, 479]):
        q = rng.normal(size=(B, H * hd)).astype(np.float32)
        qd.copy_(torch.from_numpy(q))
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        for g, out in zip(graphs, outs):
            out.fill_(9.0)
            g.replay()
            _check(torch, pool, q, n, H, host(out), tabs)


def test_attention_on_two_streams(cuda):
    torch = cuda
    H, KV, hd, page, B = 32, 8, 128, 64, 4
    rng = np.random.default_rng(13)
    pages, table = _table(rng, B, 20)
    pool = P.Pool(torch, pages, page, KV, hd, table)
    for b in range(B):
        pool.put_random(rng, b, 1280)
    q = [rng.normal(size=(B, H * hd)).astype(np.float32) for _ in range(2)]
    lens = [[1280, 3, 700, 64], [1, 1280, 1279, 0]]
    qd = [dev(torch, x) for x in q]
    ld = [dev(torch, np.array(x, np.int32)) for x in lens]
    outs = [torch.zeros(B, H * hd, device="cuda") for _ in range(2)]
    works = [P.workspace(torch, B, H, KV, hd) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for i in range(2):
            _capi.check(P.attend(torch, pool, qd[i], outs[i], H, ld[i], work=works[i], stream=streams[i].cuda_stream))
    torch.cuda.synchronize()
    for i in range(2):
        _check(torch, pool, q[i], lens[i], H, host(outs[i]))


def test_offsets_past_32_bits(cuda):
    """A pool of more than 2^31 bytes: rows at its end are written, read and attended over."""
    torch = cuda
    H, KV, hd, page = 8, 4, 128, 64
    pages = (1 << 31) // (page * KV * hd) + 40
    table = np.array([[pages - 1, 0, pages - 3], [1, pages - 2, 2]], np.int32)
    pool = P.Pool(torch, pages, page, KV, hd, table)
    rng = np.random.default_rng(1)
    n = [190, 150]
    seq = np.repeat([0, 1], n).astype(np.int32)
    pos = np.concatenate([np.arange(m) for m in n]).astype(np.int32)
    x = rng.normal(size=(len(seq), 2 * KV * hd)).astype(np.float32)
    xd, seqd, posd = dev(torch, x), dev(torch, seq), dev(torch, pos)
    _capi.check(_append(torch, pool, xd.data_ptr(), xd.data_ptr() + 4 * KV * hd, 2 * KV * hd, len(seq), seqd, posd))
    kq, ks = P.quantise(x[:, : KV * hd].astype(np.float64).reshape(-1, KV, hd))
    vq, vs = P.quantise(x[:, KV * hd:].astype(np.float64).reshape(-1, KV, hd))
    for b, off in ((0, 0), (1, n[0])):
        k, kk, v, vv = pool.rows(b, n[b])
        assert np.array_equal(k, kq[off: off + n[b]]) and np.array_equal(v, vq[off: off + n[b]])
        assert np.array_equal(kk, ks[off: off + n[b]]) and np.array_equal(vv, vs[off: off + n[b]])
    back = torch.zeros(len(seq), 2 * KV * hd, device="cuda")
    _capi.check(_read(torch, pool, back.data_ptr(), back.data_ptr() + 4 * KV * hd, 2 * KV * hd, len(seq), seqd, posd))
    want = np.concatenate([(kq * ks[..., None]).reshape(-1, KV * hd), (vq * vs[..., None]).reshape(-1, KV * hd)], 1)
    assert np.array_equal(host(back), want.astype(np.float32))
    q = rng.normal(size=(2, H * hd)).astype(np.float32)
    out = torch.empty(2, H * hd, device="cuda")
    _capi.check(P.attend(torch, pool, dev(torch, q), out, H, dev(torch, np.array(n, np.int32)),
                         work=P.workspace(torch, 2, H, KV, hd)))
    _check(torch, pool, q, n, H, host(out))


# ---- together ----------------------------------------------------------------

def test_decode_steps_of_ragged_sequences(cuda):
    """Prompts of three sequences in one append, then steps of append, attention and a batched pick:
    the cache's bytes and the attention rows equal jyc_rope_pos + jyc_attention_q8 on each sequence's
    own contiguous cache, and the picks follow the logits that the step made."""
    torch = cuda
    lib = _capi.load()
    H, KV, hd, page, V, D = 8, 2, 64, 16, 1000, 96
    rng = np.random.default_rng(21)
    B, prompts, steps = 3, [5, 40, 17], 6
    width = 5
    pages, table = _table(rng, B, width)
    pool = P.Pool(torch, pages, page, KV, hd, table)
    c, s = P.tables(width * page, hd)
    cos, sin = dev(torch, c), dev(torch, s)
    cap = width * page
    flat = [[torch.zeros(cap * KV * hd, dtype=torch.int8, device="cuda"), torch.zeros(cap * KV, device="cuda"),
             torch.zeros(cap * KV * hd, dtype=torch.int8, device="cuda"), torch.zeros(cap * KV, device="cuda")]
            for _ in range(B)]
    qw, kw = H * hd, KV * hd
    W = dev(torch, (rng.normal(size=(qw + 2 * kw, D)) / np.sqrt(D)).astype(np.float32))  # fused q|k|v rows
    head = dev(torch, (rng.normal(size=(V, qw)) / 4).astype(np.float32))
    emb = dev(torch, rng.normal(size=(V, D)).astype(np.float32))
    ld = qw + 2 * kw

    def project(x):
        y = torch.empty(x.shape[0], ld, device="cuda")
        _capi.check(lib.jyc_matmul_f32(x.data_ptr(), W.data_ptr(), y.data_ptr(), x.shape[0], ld, D, _stream(torch)))
        return y

    def contiguous(b, y, start):
        """The same rows through the one-sequence operators; returns the attention rows."""
        n = y.shape[0]
        q, k, v = (t.contiguous() for t in (y[:, :qw], y[:, qw: qw + kw], y[:, qw + kw:]))
        for t, heads in ((q, H), (k, KV)):
            _capi.check(lib.jyc_rope_pos(t.data_ptr(), n, start, heads, hd, cos.data_ptr(), sin.data_ptr(),
                                         _stream(torch)))
        o = torch.empty(n, qw, device="cuda")
        f = flat[b]
        _capi.check(lib.jyc_attention_q8(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), n, start, H, KV, hd,
                                         f[0].data_ptr(), f[1].data_ptr(), f[2].data_ptr(), f[3].data_ptr(), cap,
                                         _stream(torch)))
        return o

    ids = [rng.integers(0, V, n) for n in prompts]
    seq = dev(torch, np.repeat(np.arange(B), prompts).astype(np.int32))
    pos = dev(torch, np.concatenate([np.arange(n) for n in prompts]).astype(np.int32))
    y = project(emb[torch.from_numpy(np.concatenate(ids)).cuda()].contiguous())
    _capi.check(_append(torch, pool, y.data_ptr() + 4 * qw, y.data_ptr() + 4 * (qw + kw), ld, y.shape[0], seq, pos,
                        cos, sin))
    at = 0
    for b in range(B):
        contiguous(b, y[at: at + prompts[b]], 0)
        at += prompts[b]
    lens = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    token = torch.tensor([i[-1] for i in ids], dtype=torch.int32, device="cuda")
    work = P.workspace(torch, B, H, KV, hd)
    T = torch.tensor([0.0, 0.8, 1.2], device="cuda")
    top_k = torch.tensor([0, 20, 0], dtype=torch.int32, device="cuda")
    top_p = torch.tensor([1.0, 0.95, 0.9], device="cuda")
    for step in range(steps):
        y = project(emb[token.long()].contiguous())
        _capi.check(_append(torch, pool, y.data_ptr() + 4 * qw, y.data_ptr() + 4 * (qw + kw), ld, B, None, lens,
                            cos, sin))
        lens += 1
        out = torch.empty(B, qw, device="cuda")
        _capi.check(P.attend(torch, pool, y, out, H, lens, cos, sin, work))
        logits = torch.empty(B, V, device="cuda")
        _capi.check(lib.jyc_matmul_f32(out.data_ptr(), head.data_ptr(), logits.data_ptr(), B, V, qw, _stream(torch)))
        u = torch.from_numpy(rng.random(B).astype(np.float32)).cuda()
        probs = torch.empty(B, device="cuda")
        _capi.check(lib.jyc_sample_batch(logits.data_ptr(), V, B, V, T.data_ptr(), top_k.data_ptr(), top_p.data_ptr(),
                                         None, u.data_ptr(), token.data_ptr(), probs.data_ptr(), _stream(torch)))
        n = host(lens)
        for b in range(B):
            o = host(contiguous(b, y[b: b + 1], int(n[b]) - 1))[0]
            k8, ks, v8, vs = (host(t) for t in flat[b])
            m = int(n[b])
            pk, pks, pv, pvs = pool.rows(b, m)
            assert np.array_equal(pk.ravel(), k8[: m * kw]) and np.array_equal(pv.ravel(), v8[: m * kw])
            assert np.array_equal(pks.ravel(), ks[: m * KV]) and np.array_equal(pvs.ravel(), vs[: m * KV])
            tol = 2 * P.attention_tolerance(m, 20.0, np.abs(pv * pvs[..., None]).max())  # both sides round
            assert np.abs(host(out)[b] - o).max() <= tol
            ok = P.picks(host(logits)[b], float(T[b]), int(top_k[b]), float(top_p[b]), None, float(u[b]))
            assert int(token[b]) in ok, (step, b)


def test_error_word_reset_loses_nothing(cuda):
    """A flag raised by a call that is issued right after a reset, on a stream that the default one does not
    order, is still there to be read, while another thread keeps the default stream busy."""
    import threading
    torch = cuda
    lib = _capi.load()
    pool = P.Pool(torch, 2, 8, 1, 64, [[0, 99]])
    x = torch.zeros(1, 64, device="cuda")
    seq = torch.zeros(1, dtype=torch.int32, device="cuda")
    far, bad = (torch.tensor([p], dtype=torch.int32, device="cuda") for p in (16, 8))
    stream = torch.cuda.Stream()

    def append(pos, s):
        _capi.check(lib.jyc_kv_append_paged_q8(
            P.ptr(x), P.ptr(x), 64, 1, 1, 64, P.ptr(seq), P.ptr(pos), P.ptr(pool.table), 2, 1, None, None, 0,
            C.byref(pool.desc), s))

    big = torch.zeros(1 << 26, device="cuda")
    ends = threading.Event()

    def work():
        done = [torch.cuda.Event() for _ in range(8)]  # eight passes ahead
        for i in range(1 << 20):
            done[i % 8].synchronize()
            if ends.is_set():
                break
            big.add_(1.0)
            done[i % 8].record()

    torch.cuda.synchronize()
    other = threading.Thread(target=work)
    other.start()
    try:
        for i in range(300):
            append(far, stream.cuda_stream)             # out of range: bit 1
            assert lib.jyc_paged_error(1) == 1, i
            append(bad, stream.cuda_stream)             # a bad page: bit 2
            stream.synchronize()
            assert lib.jyc_paged_error(1) == 2, i
            assert lib.jyc_paged_error(0) == 0, i
    finally:
        ends.set()
        other.join()
