"""The paged 4-bit cache on the device (jyc_kv_append_paged_q4, jyc_kv_read_paged_q4,
jyc_attention_paged_q4, jyc_kv_evict_paged_q4) against the plain 64-bit forms of _paged4.py.

Bytes, parameters, read-back values and what an eviction keeps are equal bit for bit; attention and
the weights that it leaves are within the rounding bounds that _paged4.py derives.
"""
import numpy as np
import pytest

import _paged as P
import _paged4 as P4
from _util import dev, host
from jieyu_b200 import _capi

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_error_left(cuda):
    lib = _capi.load()
    lib.jyc_paged_error(1)
    yield
    assert lib.jyc_paged_error(1) == 0


def _table(rng, seqs, width, spare=3):
    pages = seqs * width + spare
    return pages, rng.permutation(pages)[: seqs * width].reshape(seqs, width)


def _ints(torch, x):
    return dev(torch, np.asarray(x).astype(np.int32))


# ---- append and read ---------------------------------------------------------

APPEND = [  # kv, hd, page, heads_first, rot, halves, extra floats of a row, gap, offset of K in floats
    (2, 64, 16, False, 64, False, 0, 0, 0),
    (8, 128, 32, True, 128, True, 8, 0, 0),
    (3, 80, 7, False, 80, True, 3, 1, 0),
    (1, 4, 1, True, 4, False, 0, 0, 1),
    (5, 36, 257, False, 0, False, 0, 2, 2),
    (2, 256, 16, True, 128, False, 4, 0, 0),
    (4, 132, 5, False, 66, True, 0, 0, 0),
    (16, 96, 64, True, 90, False, 0, 1, 4),
    (3, 160, 8, False, 160, True, 0, 0, 0),
    (6, 32, 9, False, 6, True, 0, 0, 0),
]


@pytest.mark.parametrize("kv,hd,page,hf,rot,halves,extra,gap,off", APPEND)
@pytest.mark.parametrize("rows", [1, 37, 300])
def test_append_and_read_back(cuda, kv, hd, page, hf, rot, halves, extra, gap, off, rows):
    torch = cuda
    rng = np.random.default_rng(rows * 1000 + hd)
    seqs = min(rows, 5)
    width = (rows + 9) // page + 1
    pages, table = _table(rng, seqs, width)
    pool = P4.Pool(torch, pages, page, kv, hd, table, hf, gap, fill=77)
    seq = np.arange(rows) % seqs
    pos = np.arange(rows) // seqs + rng.integers(0, 5)
    pad = rng.random(rows) < 0.2
    pos[pad] = -1 - rng.integers(0, 5, pad.sum())
    ld = 2 * kv * hd + extra
    x = rng.normal(size=rows * ld + off).astype(np.float32)
    if rows > 8:
        r = x[off:].reshape(rows, ld)
        r[1, : kv * hd] = 0.0                    # step and low 0
        r[2, : kv * hd] = 1e-9                   # step 0 in fp16
        r[3, hd // 2] = 3e38                     # beyond fp16: held
        r[4, :hd] *= np.float32(1e-5)            # steps below fp16's normal numbers
        r[5, kv * hd:] = 40000.0 * np.sign(r[5, kv * hd:])
        r[6, kv * hd:] = 1000.0                  # all values alike
        r[7, -hd - extra: -extra or None] += 300.0
    cos = sin = rp = None
    turn = pos
    if rot:
        n = width * page + 40
        cos, sin = P.tables(n, rot)
        c, s = dev(torch, cos), dev(torch, sin)
        rp = P4.rope(c, s, halves)
        if rows == 37:
            turn = rng.integers(0, n, rows)
    xd, seqd, posd = dev(torch, x), _ints(torch, seq), _ints(torch, pos)
    turnd = None if turn is pos else _ints(torch, turn)
    base = xd.data_ptr() + 4 * off
    before = [host(t).copy() for t in (pool.k, pool.v, pool.kp, pool.vp, pool.mass)]
    _capi.check(P4.append(torch, pool, base, base + 4 * kv * hd, ld, rows, seqd, posd, rp, turnd))
    body = x[off:].reshape(rows, ld).astype(np.float64)
    K = body[:, : kv * hd].reshape(rows, kv, hd)
    V = body[:, kv * hd: 2 * kv * hd].reshape(rows, kv, hd)
    live = pos >= 0
    if rot:
        K = K.copy()
        K[live] = P4.turn(K[live], turn[live], cos, sin, halves)
    (kq, kst, klo), (vq, vst, vlo) = P4.quantise(K), P4.quantise(V)
    wk, wv, wkp, wvp, wm = before
    G = pool.G
    for i in np.flatnonzero(live):
        at = pool.where(seq[i], pos[i])
        wk[at][:, : 16 * G], wv[at][:, : 16 * G] = P4.pack(kq[i]), P4.pack(vq[i])
        wkp[at][:, :G], wvp[at][:, :G] = P4.params(kst[i], klo[i]), P4.params(vst[i], vlo[i])
        wm[at] = 0.0
    for t, want in ((pool.k, wk), (pool.v, wv), (pool.kp, wkp), (pool.vp, wvp), (pool.mass, wm)):
        assert np.array_equal(host(t), want)
    back = torch.full((rows * ld + off,), -7.0, device="cuda")
    bb = back.data_ptr() + 4 * off
    _capi.check(P4.read(torch, pool, bb, bb + 4 * kv * hd, ld, rows, seqd, posd))
    got = host(back)
    want = np.full((rows, ld), -7.0, np.float32)
    want[live, : kv * hd] = P4.values(kq, kst, klo)[live].reshape(-1, kv * hd).astype(np.float32)
    want[live, kv * hd: 2 * kv * hd] = P4.values(vq, vst, vlo)[live].reshape(-1, kv * hd).astype(np.float32)
    assert np.all(got[:off] == -7.0)
    assert np.array_equal(got[off:].reshape(rows, ld), want)


def test_values_that_are_not_numbers(cuda):
    torch = cuda
    rng = np.random.default_rng(3)
    kv, hd, n = 3, 72, 9
    x = rng.normal(size=(n, kv, hd)).astype(np.float32)
    x[1, 0, 3] = np.inf
    x[2, 1, 5] = np.nan
    x[3, 2] = -np.inf
    x[4, 0] = np.nan
    x[5, 1, 40] = -np.inf
    x[6, 2, 64:] = np.nan
    x[7, 0, 0], x[7, 0, 1] = 3e38, -3e38
    pool = P4.Pool(torch, 1, n, kv, hd, [[0]], fill=9, mass=False)
    xd = dev(torch, x)
    pos, seq = _ints(torch, np.arange(n)), _ints(torch, np.zeros(n))
    _capi.check(P4.append(torch, pool, xd.data_ptr(), xd.data_ptr(), kv * hd, n, seq, pos))
    q, st, lo = P4.quantise(x.astype(np.float64))
    for b, p in ((pool.k, pool.kp), (pool.v, pool.vp)):
        assert np.array_equal(host(b)[0], P4.pack(q)) and np.array_equal(host(p)[0], P4.params(st, lo))
    assert np.isfinite(host(pool.kp).astype(np.float32)).all()


def test_append_and_read_skip_what_is_out_of_range(cuda):
    torch = cuda
    lib = _capi.load()
    kv, hd, page = 2, 64, 8
    table = np.array([[0, 1], [2, 99], [3, -5]])
    pool = P4.Pool(torch, 6, page, kv, hd, table, fill=3)
    before = host(pool.k).copy()
    x = torch.randn(6, kv * hd, device="cuda")
    cos, sin = P.tables(12, hd)
    c, s = dev(torch, cos), dev(torch, sin)
    cases = [  # sequences, positions, rope, rope positions, error bits
        ([0, 0], [16, 100], None, None, 1), ([3, -1], [0, 0], None, None, 1), ([1, 2], [8, 9], None, None, 2),
        ([0, 1], [12, 13], P4.rope(c, s, True), None, 4), ([0, 1], [1, 2], P4.rope(c, s, False), [-1, 12], 4),
        ([0, 1], [1, 2], P4.rope(c, s, False, 1), None, 4)]
    for seq, pos, rp, turn, bits in cases:
        n = len(seq)
        args = (_ints(torch, seq), _ints(torch, pos))
        _capi.check(P4.append(torch, pool, x.data_ptr(), x.data_ptr(), kv * hd, n, *args, rp,
                              None if turn is None else _ints(torch, turn)))
        assert lib.jyc_paged_error(1) & ~2 == bits & ~2 and np.array_equal(host(pool.k), before)
        if rp is None:
            y = torch.full((n, 2 * kv * hd), 4.0, device="cuda")
            _capi.check(P4.read(torch, pool, y.data_ptr(), y.data_ptr() + 4 * kv * hd, 2 * kv * hd, n, *args))
            assert lib.jyc_paged_error(1) == bits and np.all(host(y) == 4.0)


# ---- attention ---------------------------------------------------------------

def _check(torch, rng, pool, q, out, mass0, H, lens, cos=None, sin=None, halves=False, turn=None):
    """Rows of out, and the masses where the pool has them, against the 64-bit form."""
    hd, kv, G = pool.hd, pool.kv, pool.G
    got, n = host(out), np.asarray(lens)
    x = host(q).astype(np.float64)[:, : H * hd].reshape(len(n), H, hd)
    worst = 0.0
    for b in range(len(n)):
        if n[b] <= 0:
            assert np.all(got[b, : H * hd] == 0.0)
            continue
        qb = x[b: b + 1]
        if cos is not None:
            qb = P4.turn(qb, np.array([n[b] - 1 if turn is None else turn[b]]), cos, sin, halves)
        qi, qs = P.quantise(qb[0])
        kq, kst, klo, vq, vst, vlo = pool.rows(b, n[b])
        want, mass = P4.attention(qi, qs, P4.values(kq, kst, klo), P4.values(vq, vst, vlo))
        smax = P4.magnitudes(qi, qs, kst, klo, hd)
        vmax = (np.abs(vlo) + 15 * vst).max()
        tol = P4.out_tolerance(n[b], G, smax, vmax)
        err = np.abs(got[b, : H * hd].reshape(H, hd) - want).max()
        assert err <= tol, (b, n[b], err, tol)
        worst = max(worst, err / tol)
        if pool.mass is not None:
            was = mass0[b][: n[b]]
            now = pool.masses(b, n[b]).astype(np.float64)
            rel = P4.rounding(n[b], G, smax, H // kv)
            # one more rounding as the weight is added to what was there; weights below 2^-126 may be lost
            assert np.all(np.abs(now - was - mass) <= mass * rel + P.U24 * (was + mass) + H * 2.0 ** -125), b
    return worst


ATTENTION = [  # H, kv, hd, page, heads_first, rot, halves, gap, lens
    (14, 2, 64, 16, False, 64, True, 0, [513]),
    (1, 1, 4, 1, False, 0, False, 0, [1, 2, 33]),
    (4, 4, 128, 64, True, 128, False, 0, [1, 0, 64, 65, 200, 1000]),
    (32, 8, 128, 32, False, 64, True, 0, [31, 32, 33, 700, 0, 0, 5]),
    (12, 3, 80, 7, False, 80, True, 1, [1, 7, 8, 100, 641]),
    (16, 1, 64, 128, False, 0, False, 0, [300, 1]),
    (24, 1, 96, 16, True, 96, False, 2, [90, 1500, 3]),
    (40, 2, 36, 257, False, 30, True, 0, [600, 258]),
    (8, 8, 256, 16, True, 256, True, 0, [17, 150, 0, 33]),
    (20, 4, 132, 5, False, 0, False, 0, [44, 1, 999]),
    (48, 2, 160, 32, False, 80, False, 0, [129, 64]),
    (9, 3, 192, 48, False, 192, True, 0, [200, 1, 1]),
    (6, 6, 32, 3, True, 0, False, 0, [3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13]),
    (7, 1, 128, 64, False, 128, True, 0, [4100]),
    (25, 1, 64, 64, True, 64, True, 0, [2050, 31]),
]


@pytest.mark.parametrize("H,kv,hd,page,hf,rot,halves,gap,lens", ATTENTION)
@pytest.mark.parametrize("mass", [False, True])
def test_attention(cuda, H, kv, hd, page, hf, rot, halves, gap, lens, mass):
    torch = cuda
    rng = np.random.default_rng(H * 100 + hd)
    seqs, width = len(lens), max(lens) // page + 2
    pages, table = _table(rng, seqs, width)
    pool = P4.Pool(torch, pages, page, kv, hd, table, hf, gap, mass=mass)
    pool.put_random(rng, lens)
    mass0 = None
    if mass:
        pool.mass.uniform_(0.0, 2.0)
        before = host(pool.mass).copy()
        mass0 = [pool.masses(b, width * page).astype(np.float64) for b in range(seqs)]
    cos = sin = rp = turn = None
    if rot:
        cos, sin = P.tables(max(lens) + 20, rot)
        c, s = dev(torch, cos), dev(torch, sin)
        rp = P4.rope(c, s, halves)
        if H % 2 == 0:  # positions apart from the lengths
            turn = np.minimum(np.array(lens) + rng.integers(0, 10, seqs), max(lens) + 19)
    ldq = H * hd + 4 * (H % 3)
    q, out = 2 * torch.randn(seqs, ldq, device="cuda"), torch.full((seqs, H * hd + 3), 8.0, device="cuda")
    lensd = _ints(torch, lens)
    work = P4.workspace(torch, seqs, H, kv, hd, width * page if mass else 0)
    _capi.check(P4.attend(torch, pool, q, out, H, lensd, rp, None if turn is None else _ints(torch, turn), work))
    _check(torch, rng, pool, q, out, mass0, H, lens, cos, sin, halves, turn)
    assert np.all(host(out)[:, H * hd:] == 8.0)
    if mass:  # places that no key holds stay as they were
        now = host(pool.mass)
        for b in range(seqs):
            for j in range(lens[b]):
                at = pool.where(b, j)
                before[at] = now[at]
        assert np.array_equal(now, before)


# tensor copies of every row size and page, with gaps; head counts that teams of warps divide and do not
COPIES = [  # H, kv, hd, page, heads_first, gap, lens
    (32, 8, 128, 32, False, 1, [700, 64, 1]), (12, 6, 128, 16, False, 0, [1000, 17, 16]), (5, 5, 128, 64, False, 3, [333]),
    (64, 16, 128, 64, True, 0, [129, 0, 2000]), (24, 12, 64, 32, False, 2, [95, 4000]), (8, 8, 64, 16, True, 0, [1, 15, 16, 17]),
    (36, 3, 64, 64, False, 0, [65, 1300]), (72, 4, 128, 128, False, 0, [640, 1]), (30, 10, 256, 16, False, 1, [70, 500]),
    (9, 9, 160, 8, True, 0, [260]), (14, 7, 100, 64, False, 0, [128, 3000]), (4, 2, 48, 32, False, 0, [33, 77]),
]


@pytest.mark.parametrize("H,kv,hd,page,hf,gap,lens", COPIES)
def test_attention_by_every_copy(cuda, H, kv, hd, page, hf, gap, lens):
    torch = cuda
    rng = np.random.default_rng(H + hd)
    pages, table = _table(rng, len(lens), max(lens) // page + 1)
    pool = P4.Pool(torch, pages, page, kv, hd, table, hf, gap, fill=255)
    pool.kp.fill_(float("nan"))  # rows that no length reaches, and gaps, hold NaN
    pool.vp.fill_(float("inf"))
    pool.mass.zero_()
    filled = P4.Pool(torch, pages, page, kv, hd, table, hf, gap)
    filled.put_random(rng, lens)
    for b, n in enumerate(lens):
        for j in range(n):
            at = pool.where(b, j)
            for x, y, w in ((pool.k, filled.k, 16 * pool.G), (pool.v, filled.v, 16 * pool.G), (pool.kp, filled.kp, pool.G),
                            (pool.vp, filled.vp, pool.G)):
                x[at][:, :w] = y[at][:, :w]
    q, out = torch.randn(len(lens), H * hd, device="cuda"), torch.full((len(lens), H * hd), 8.0, device="cuda")
    work = P4.workspace(torch, len(lens), H, kv, hd, table.shape[1] * page)
    _capi.check(P4.attend(torch, pool, q, out, H, _ints(torch, lens), work=work))
    _check(torch, rng, pool, q, out, [np.zeros((n, kv)) for n in lens], H, lens)


def test_many_short_sequences(cuda):
    """More sequences than a CTA has threads, most of them short or empty."""
    torch = cuda
    rng = np.random.default_rng(44)
    kv, hd, H, page, seqs = 2, 64, 4, 16, 900
    lens = rng.integers(0, 40, seqs)
    lens[rng.random(seqs) < 0.3] = 0
    lens[17] = 3000
    pages, table = 3 * seqs + 188, np.zeros((seqs, 188), np.int64)
    order = rng.permutation(pages)
    table[:, :3] = order[: 3 * seqs].reshape(seqs, 3)
    table[17] = order[3 * seqs:]
    pool = P4.Pool(torch, pages, page, kv, hd, table)
    pool.put_random(rng, None)
    q, out = torch.randn(seqs, H * hd, device="cuda"), torch.full((seqs, H * hd), 8.0, device="cuda")
    _capi.check(P4.attend(torch, pool, q, out, H, _ints(torch, lens)))
    _check(torch, rng, pool, q, out, [np.zeros((max(n, 0), kv)) for n in lens], H, lens)


def test_attention_without_a_workspace_and_again(cuda):
    """Scratch in stream order; a second call gives the same bits, and the masses twice the weight."""
    torch = cuda
    rng = np.random.default_rng(5)
    lens = [900, 1, 0, 333]
    pages, table = _table(rng, 4, 30)
    pool = P4.Pool(torch, pages, 32, 2, 128, table)
    pool.put_random(rng, lens)
    q = torch.randn(4, 8 * 128, device="cuda")
    outs = [torch.zeros(4, 8 * 128, device="cuda") for _ in range(3)]
    masses = []
    for out in outs:
        _capi.check(P4.attend(torch, pool, q, out, 8, _ints(torch, lens)))
        masses.append(host(pool.mass).copy())
    assert np.array_equal(host(outs[0]), host(outs[1])) and np.array_equal(host(outs[0]), host(outs[2]))
    assert np.array_equal(masses[1], 2 * masses[0])
    pool.mass.copy_(torch.from_numpy(masses[0]))
    _check(torch, rng, pool, q, outs[0], [np.zeros((n, 2)) for n in lens], 8, lens)


@pytest.mark.parametrize("H,kv,hd,page", [(8, 2, 128, 64), (12, 1, 64, 16), (4, 4, 96, 5), (3, 1, 256, 32)])
@pytest.mark.parametrize("scale", [1e-4, 1.0, 3000.0])
def test_steps_of_every_size(cuda, H, kv, hd, page, scale):
    """V far smaller and far larger than 1, K moderate, some keys of one size and some of another."""
    torch = cuda
    rng = np.random.default_rng(6)
    lens = [70, 400]
    pages, table = _table(rng, 2, -(-400 // page) + 1)
    pool = P4.Pool(torch, pages, page, kv, hd, table, mass=False)
    pool.put_random(rng, lens)
    pool.vp.mul_(scale)
    pool.vp[::3].mul_(0.01)
    pool.kp.mul_(0.3)
    q = torch.randn(2, H * hd, device="cuda")
    out = torch.zeros(2, H * hd, device="cuda")
    _capi.check(P4.attend(torch, pool, q, out, H, _ints(torch, lens)))
    _check(torch, rng, pool, q, out, None, H, lens)


@pytest.mark.parametrize("H,kv,hd,page,n", [(32, 8, 128, 64, 5000), (14, 2, 64, 16, 513), (8, 8, 64, 32, 3000),
                                            (16, 1, 128, 32, 700), (6, 2, 80, 7, 900), (24, 1, 256, 16, 400),
                                            (5, 5, 192, 64, 2000)])
def test_attention_is_as_close_as_plain_fp32(cuda, H, kv, hd, page, n):
    """The tolerance above is for roundings that all fall the same way. In the root mean square the result is no further from
    the 64-bit one than four times what elementary fp32 operations are, and 2^-21 of its own size (weights as two halves)."""
    torch = cuda
    rng = np.random.default_rng(62)
    pages, table = _table(rng, 1, n // page + 1)
    pool = P4.Pool(torch, pages, page, kv, hd, table, mass=False)
    pool.put_random(rng, [n])
    q, out = 2 * torch.randn(1, H * hd, device="cuda"), torch.zeros(1, H * hd, device="cuda")
    _capi.check(P4.attend(torch, pool, q, out, H, _ints(torch, [n])))
    qi, qs = P.quantise(host(q).astype(np.float64).reshape(H, hd))
    kq, kst, klo, vq, vst, vlo = pool.rows(0, n)
    k, v = P4.values(kq, kst, klo), P4.values(vq, vst, vlo)
    want, _ = P4.attention(qi, qs, k, v)
    t = lambda x: torch.from_numpy(x.astype(np.float32)).cuda()  # noqa: E731
    group = H // kv
    s = torch.einsum("hgd,nhd->hgn", t(qi).reshape(kv, group, hd), t(k)) * (t(qs) / hd ** 0.5).reshape(kv, group, 1)
    p = (s - s.amax(-1, keepdim=True)).exp()
    plain = host(torch.einsum("hgn,nhd->hgd", p / p.sum(-1, keepdim=True), t(v)).reshape(H, hd)).astype(np.float64)
    size = lambda x: np.sqrt(np.mean(x ** 2))  # noqa: E731
    off = size(host(out).reshape(H, hd) - want)
    assert off <= 4 * size(plain - want) + 2.0 ** -21 * size(want), (off / size(want), size(plain - want) / size(want))


def test_parameters_of_either_sign(cuda):
    """Values are low + step * q whatever the signs: rows that this library did not write."""
    torch = cuda
    rng = np.random.default_rng(61)
    for H, kv, hd, page in ((8, 2, 128, 64), (12, 2, 64, 32), (3, 1, 192, 16)):
        lens = [300, 65]
        pages, table = _table(rng, 2, 300 // page + 1)
        pool = P4.Pool(torch, pages, page, kv, hd, table)
        pool.put_random(rng, lens)
        for p in (pool.kp, pool.vp):
            p.mul_(torch.from_numpy(rng.choice([-1.0, 1.0, 3.0, -0.01], tuple(p.shape))).cuda().half())
        q, out = torch.randn(2, H * hd, device="cuda"), torch.zeros(2, H * hd, device="cuda")
        _capi.check(P4.attend(torch, pool, q, out, H, _ints(torch, lens)))
        _check_signed(torch, pool, q, out, H, lens)


def _check_signed(torch, pool, q, out, H, lens):
    x = host(q).astype(np.float64).reshape(len(lens), H, pool.hd)
    for b, n in enumerate(lens):
        qi, qs = P.quantise(x[b])
        kq, kst, klo, vq, vst, vlo = pool.rows(b, n)
        want, _ = P4.attention(qi, qs, P4.values(kq, kst, klo), P4.values(vq, vst, vlo))
        tol = P4.out_tolerance(n, pool.G, P4.magnitudes(qi, qs, np.abs(kst), klo, pool.hd), (np.abs(vlo) + 15 * np.abs(vst)).max())
        assert np.abs(host(out)[b].reshape(H, pool.hd) - want).max() <= tol


def test_equal_and_extreme_scores(cuda):
    """Rows whose keys are all alike (weights 1 / n), and one key that takes all of the weight."""
    torch = cuda
    rng = np.random.default_rng(7)
    lens, kv, hd, H, page = [257, 257, 129], 2, 64, 8, 16
    pages, table = _table(rng, 3, 17)
    pool = P4.Pool(torch, pages, page, kv, hd, table)
    pool.put_random(rng, lens)
    for b in (0, 1):
        for j in range(lens[b]):
            at = pool.where(b, j)
            pool.kp[at] = 0.0 if b == 0 else 1e-3
    j = 200
    pool.k[pool.where(1, j)] = 255
    pool.kp[pool.where(1, j)] = 200.0
    q = torch.randn(3, H * hd, device="cuda").abs()
    out = torch.zeros(3, H * hd, device="cuda")
    _capi.check(P4.attend(torch, pool, q, out, H, _ints(torch, lens)))
    _check(torch, rng, pool, q, out, [np.zeros((n, kv)) for n in lens], H, lens)
    m = pool.masses(1, 257)
    assert np.all(m[j] == H / kv) and np.all(np.delete(m, j, 0) == 0.0)
    assert np.allclose(pool.masses(0, 257), 4 / 257, rtol=1e-5, atol=0)


def test_parameters_that_are_not_numbers(cuda):
    """A key whose parameters are infinite or NaN makes its kv head's rows NaN and no others; behind the length it
    does nothing."""
    torch = cuda
    rng = np.random.default_rng(8)
    kv, hd, H, page = 2, 128, 8, 32
    for name in ("kp", "vp"):
        for value in (float("inf"), float("-inf"), float("nan")):
            for part in (0, 1):
                lens = [100, 60]
                pages, table = _table(rng, 2, 5)
                pool = P4.Pool(torch, pages, page, kv, hd, table, mass=False)
                pool.put_random(rng, lens)
                getattr(pool, name)[pool.where(0, 37, 1)][2, part] = value
                getattr(pool, name)[pool.where(1, 60, 0)][0, part] = value
                getattr(pool, name)[pool.where(1, 95, 1)][3, part] = value
                q, out = torch.randn(2, H * hd, device="cuda"), torch.zeros(2, H * hd, device="cuda")
                _capi.check(P4.attend(torch, pool, q, out, H, _ints(torch, lens)))
                got = host(out).reshape(2, H, hd)
                bad = got[0, H // 2:]
                assert np.isnan(bad).all(), (name, value, part)
                assert np.isfinite(got[0, : H // 2]).all() and np.isfinite(got[1]).all()


def test_lengths_and_pages_out_of_range(cuda):
    torch = cuda
    lib = _capi.load()
    rng = np.random.default_rng(9)
    kv, hd, H, page = 2, 64, 4, 16
    pages, table = _table(rng, 4, 4)
    table[1, 2] = pages + 7
    table[2, 0] = -3
    pool = P4.Pool(torch, pages, page, kv, hd, table)
    pool.put_random(rng, None)
    q, out = torch.randn(4, H * hd, device="cuda"), torch.full((4, H * hd), 9.0, device="cuda")
    cos, sin = P.tables(50, hd)
    c, s = dev(torch, cos), dev(torch, sin)
    # a length beyond the table is cut to it
    _capi.check(P4.attend(torch, pool, q, out, H, _ints(torch, [900, 30, 0, -4]), seqs=4))
    assert lib.jyc_paged_error(1) == 1
    zero = [np.zeros((64, kv))] * 4
    _check(torch, rng, pool, q, out, zero, H, [64, 30, 0, 0])
    # keys of pages that are not there weigh nothing
    pool.mass.zero_()
    _capi.check(P4.attend(torch, pool, q, out, H, _ints(torch, [10, 60, 40, 16])))
    assert lib.jyc_paged_error(1) == 2
    got = host(out)
    for b, n, gone in ((1, 60, range(32, 48)), (2, 40, range(0, 16))):
        table_b = table.copy()
        table_b[b] = np.where((table_b[b] < 0) | (table_b[b] >= pages), 0, table_b[b])
        kq, kst, klo, vq, vst, vlo = pool.rows(b, n, table_b)
        keep = np.setdiff1d(np.arange(n), list(gone))
        qi, qs = P.quantise(host(q).astype(np.float64)[b].reshape(H, hd))
        want, mass = P4.attention(qi, qs, P4.values(kq, kst, klo)[keep], P4.values(vq, vst, vlo)[keep])
        tol = P4.out_tolerance(n, 2, P4.magnitudes(qi, qs, kst, klo, hd), (np.abs(vlo) + 15 * vst).max())
        assert np.abs(got[b].reshape(H, hd) - want).max() <= tol
    # query positions outside of the tables (and all keys of sequence 2 lie on a page that is not there)
    for turn, want in (([10, 50, -1, 3], (1, 2)), ([49, 2**31 - 1, 0, -7], (1, 2, 3))):
        _capi.check(P4.attend(torch, pool, q, out, H, _ints(torch, [5, 6, 7, 8]), P4.rope(c, s, True), _ints(torch, turn)))
        assert lib.jyc_paged_error(1) & 4
        got = np.abs(host(out)).sum(-1)
        assert [b for b in range(4) if got[b] == 0.0] == list(want)
        lib.jyc_paged_error(1)


def test_graph_replays_for_new_lengths(cuda):
    torch = cuda
    rng = np.random.default_rng(10)
    kv, hd, H, page, seqs = 2, 128, 8, 32, 3
    pages, table = _table(rng, seqs, 20)
    pool = P4.Pool(torch, pages, page, kv, hd, table)
    pool.put_random(rng, None)
    q, out = torch.randn(seqs, H * hd, device="cuda"), torch.zeros(seqs, H * hd, device="cuda")
    lens = _ints(torch, [1, 1, 1])
    work = P4.workspace(torch, seqs, H, kv, hd, 640)
    _capi.check(P4.attend(torch, pool, q, out, H, lens, work=work))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _capi.check(P4.attend(torch, pool, q, out, H, lens, work=work))
    for n in ([640, 3, 0], [0, 0, 0], [1, 500, 33]):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        pool.mass.zero_()
        q.normal_()
        work.fill_(255)
        graph.replay()
        _check(torch, rng, pool, q, out, [np.zeros((m, kv)) for m in n], H, n)


def test_two_streams(cuda):
    """Calls that overlap in time, each with its own workspace (or scratch), give what they give alone."""
    torch = cuda
    rng = np.random.default_rng(11)
    kv, hd, H, page = 2, 64, 8, 64
    lens = [3000, 17]
    sets = []
    for i in range(2):
        pages, table = _table(rng, 2, 48)
        pool = P4.Pool(torch, pages, page, kv, hd, table)
        pool.put_random(rng, lens)
        q = torch.randn(2, H * hd, device="cuda")
        out = torch.zeros(2, H * hd, device="cuda")
        work = P4.workspace(torch, 2, H, kv, hd, 48 * page) if i else None
        sets.append((pool, q, out, work, _ints(torch, lens), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(4):
        for pool, q, out, work, n, st in sets:
            _capi.check(P4.attend(torch, pool, q, out, H, n, work=work, stream=st.cuda_stream))
    torch.cuda.synchronize()
    for pool, q, out, work, n, st in sets:
        pool.mass.mul_(0.25)
        _check(torch, rng, pool, q, out, [np.zeros((m, kv)) for m in lens], H, lens)


def test_sequences_that_share_pages(cuda):
    """A prefix that several sequences hold: its keys gather the weight of all of them."""
    torch = cuda
    rng = np.random.default_rng(12)
    kv, hd, H, page = 1, 64, 4, 16
    table = np.array([[0, 1, 2], [0, 1, 3], [0, 1, 4]])
    pool = P4.Pool(torch, 5, page, kv, hd, table)
    pool.put_random(rng, None)
    lens = [48, 40, 33]
    q, out = torch.randn(3, H * hd, device="cuda"), torch.zeros(3, H * hd, device="cuda")
    _capi.check(P4.attend(torch, pool, q, out, H, _ints(torch, lens)))
    total = np.zeros((5 * page, kv))
    x = host(q).astype(np.float64).reshape(3, H, hd)
    rel = 0.0
    for b in range(3):
        kq, kst, klo, vq, vst, vlo = pool.rows(b, lens[b])
        qi, qs = P.quantise(x[b])
        _, mass = P4.attention(qi, qs, P4.values(kq, kst, klo), P4.values(vq, vst, vlo))
        at = table[b, np.arange(lens[b]) // page] * page + np.arange(lens[b]) % page
        total[at] += mass
        rel = max(rel, P4.rounding(lens[b], 2, P4.magnitudes(qi, qs, kst, klo, hd), H))
    got = host(pool.mass).reshape(-1, kv)
    assert np.all(np.abs(got - total) <= total * (rel + 3 * P.U24) + 2.0 ** -120)


def test_pages_beyond_32_bit_offsets(cuda):
    """Page strides that pass 2^31 bytes (and 2^31 parameters): rows of far pages are found."""
    torch = cuda
    rng = np.random.default_rng(13)
    kv, hd, H, page = 1, 64, 2, 2
    far = (1 << 31) + 32
    k, v = (torch.zeros(2 * far + 4096, dtype=torch.uint8, device="cuda") for _ in range(2))
    pool = P4.Pool(torch, 3, page, kv, hd, [[2, 0]])
    pool.put_random(rng, None)
    for i in range(3):
        for big, small in ((k, pool.k), (v, pool.v)):
            big[i * far: i * far + page * 32] = small[i].reshape(-1)
    small_k, small_v = pool.desc.k, pool.desc.v
    q, want, got = torch.randn(1, H * hd, device="cuda"), *(torch.zeros(1, H * hd, device="cuda") for _ in range(2))
    n = _ints(torch, [4])
    _capi.check(P4.attend(torch, pool, q, want, H, n))
    pool.desc.k, pool.desc.v, pool.desc.page_stride = k.data_ptr(), v.data_ptr(), far
    _capi.check(P4.attend(torch, pool, q, got, H, n))
    assert np.array_equal(host(want), host(got)) and np.abs(host(got)).sum() > 0
    seq, pos = _ints(torch, [0, 0, 0]), _ints(torch, [0, 1, 3])
    a, b = (torch.zeros(3, 2 * hd, device="cuda") for _ in range(2))
    _capi.check(P4.read(torch, pool, a.data_ptr(), a.data_ptr() + 4 * hd, 2 * hd, 3, seq, pos))
    pool.desc.k, pool.desc.v, pool.desc.page_stride = small_k, small_v, page * 32
    _capi.check(P4.read(torch, pool, b.data_ptr(), b.data_ptr() + 4 * hd, 2 * hd, 3, seq, pos))
    assert np.array_equal(host(a), host(b)) and np.abs(host(a)).sum() > 0


# ---- eviction ----------------------------------------------------------------

def _set_mass(pool, rng, lens, kind):
    m = np.exp(2 * rng.normal(size=tuple(pool.mass.shape))).astype(np.float32)
    if kind == "ties":
        m = np.float32(rng.integers(0, 4, m.shape))
    elif kind == "equal":
        m[:] = 1.5
    elif kind == "odd":
        pick = rng.random(m.shape)
        m[pick < 0.2] = np.nan
        m[(pick > 0.2) & (pick < 0.3)] = np.inf
        m[(pick > 0.3) & (pick < 0.4)] = -np.inf
        m[(pick > 0.4) & (pick < 0.5)] = 0.0
        m[(pick > 0.5) & (pick < 0.6)] = -0.0
        m[(pick > 0.6) & (pick < 0.7)] = 1e-42
        m[(pick > 0.7) & (pick < 0.8)] *= -1
    elif kind == "small":
        m *= np.float32(1e-30)
    pool.mass.copy_(pool.torch.from_numpy(m))


EVICT = [  # kv, hd, page, heads_first, gap, lens, budget, recent
    (2, 64, 16, False, 0, [300, 100, 0, 128, 129], 128, 32),
    (1, 128, 64, True, 0, [1, 2, 3, 4], 1, 0),
    (3, 80, 7, False, 1, [50, 49, 48, -3], 48, 48),
    (8, 128, 32, False, 0, [2304, 2049], 2048, 256),
    (2, 36, 257, True, 2, [1000, 257, 700], 300, 0),
    (1, 256, 5, False, 0, [5000], 17, 3),
    (4, 4, 1, True, 0, [40, 41], 40, 1),
    (2, 160, 16, False, 0, [12000, 3], 9999, 100),
    (1, 64, 64, False, 0, [70000], 1000, 64),
]


@pytest.mark.parametrize("kv,hd,page,hf,gap,lens,budget,recent", EVICT)
@pytest.mark.parametrize("kind", ["plain", "ties", "equal", "odd", "small"])
def test_eviction(cuda, kv, hd, page, hf, gap, lens, budget, recent, kind):
    torch = cuda
    rng = np.random.default_rng(budget + hd)
    seqs, width, new_width = len(lens), -(-max(lens) // page), -(-budget // page)
    pages, both = _table(rng, seqs, width + new_width)
    table, new = both[:, :width], both[:, width:]
    pool = P4.Pool(torch, pages, page, kv, hd, table, hf, gap)
    pool.put_random(rng, None)
    _set_mass(pool, rng, lens, kind)
    arrays = (pool.k, pool.v, pool.kp, pool.vp, pool.mass)
    want = [host(t).copy() for t in arrays]
    newd, new_lens = _ints(torch, new), torch.full((seqs,), 99, dtype=torch.int32, device="cuda")
    kept = torch.full((seqs, kv, budget), 99, dtype=torch.int32, device="cuda")
    lensd = _ints(torch, lens)
    _capi.check(P4.evict(torch, pool, lensd, budget, recent, newd, new_lens, kept))
    n = np.maximum(lens, 0)
    assert np.array_equal(host(new_lens), np.minimum(n, budget)) and np.array_equal(host(lensd), lens)
    wk = np.full((seqs, kv, budget), -1)
    for b in range(seqs):
        if n[b] == 0:
            continue
        m = pool.masses(b, n[b])
        for h in range(kv):
            rows = P4.kept_rows(m[:, h], n[b], budget, recent)
            wk[b, h, : len(rows)] = rows
            src = table[b, rows // page], rows % page
            dst = new[b, np.arange(len(rows)) // page], np.arange(len(rows)) % page
            s, d = ((src[0], h, src[1]), (dst[0], h, dst[1])) if hf else ((*src, h), (*dst, h))
            for t, G in zip(want, (16 * pool.G, 16 * pool.G, pool.G, pool.G, None)):
                if G is None:
                    t[d] = t[s]
                else:
                    t[(*d, slice(0, G))] = t[(*s, slice(0, G))]
    assert np.array_equal(host(kept), wk)
    for t, w in zip(arrays, want):
        assert np.array_equal(host(t), w, equal_nan=t.is_floating_point())


def test_a_sequence_within_the_budget_may_keep_its_pages(cuda):
    torch = cuda
    rng = np.random.default_rng(20)
    kv, hd, page = 2, 64, 16
    table = np.arange(8).reshape(2, 4)
    new = np.array([[0, 1, 2, 3], [8, 9, 10, 11]])
    pool = P4.Pool(torch, 12, page, kv, hd, table)
    pool.put_random(rng, None)
    _set_mass(pool, rng, None, "plain")
    before = [host(t).copy() for t in (pool.k, pool.kp, pool.v, pool.vp, pool.mass)]
    kept, nl = torch.zeros(2, kv, 60, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    _capi.check(P4.evict(torch, pool, _ints(torch, [60, 64]), 60, 10, _ints(torch, new), nl, kept))
    assert list(host(nl)) == [60, 60]
    for t, was in zip((pool.k, pool.kp, pool.v, pool.vp, pool.mass), before):
        assert np.array_equal(host(t)[:8], was[:8])


def test_eviction_with_lengths_and_pages_out_of_range(cuda):
    torch = cuda
    lib = _capi.load()
    rng = np.random.default_rng(21)
    kv, hd, page = 1, 64, 16
    table = np.array([[0, 1, 2], [3, 77, 4], [5, 6, 7]])
    new = np.array([[8, 9], [10, 11], [12, -1]])
    pool = P4.Pool(torch, 13, page, kv, hd, table)
    pool.put_random(rng, None)
    _set_mass(pool, rng, None, "plain")
    k0 = host(pool.k).copy()
    kept, nl = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((3, kv, 30), (3,)))
    _capi.check(P4.evict(torch, pool, _ints(torch, [5000, 48, 48]), 30, 4, _ints(torch, new), nl, kept))
    assert lib.jyc_paged_error(1) == 3
    assert list(host(nl)) == [30, 30, 30]
    got, rows = host(pool.k), host(kept)
    assert np.array_equal(rows[0, 0], P4.kept_rows(pool.masses(0, 48)[:, 0], 48, 30, 4))
    for b in range(3):
        for to, frm in enumerate(rows[b, 0]):
            dp, sp = new[b, to // page], table[b, frm // page]
            if dp == -1:
                continue
            want = k0[dp, to % page] if sp == 77 else k0[sp, frm % page]
            assert np.array_equal(got[dp, to % page], want)
    # rows of the page that is not there are the first to go
    assert np.intersect1d(rows[1, 0], np.arange(16, 32)).size == max(0, 30 - 32)


# ---- together ----------------------------------------------------------------

def test_a_serving_loop(cuda):
    """8-bit projections, rotary rows, append, attention with gathered weights and eviction, step after step, against
    the same steps in 64 bits (the projections' whole numbers and the stored bits are equal; only attention rounds)."""
    torch = cuda
    rng = np.random.default_rng(30)
    lib = _capi.load()
    seqs, hidden, H, kv, hd, page, budget, recent, steps = 3, 192, 4, 2, 64, 8, 24, 6, 40
    width, new_width = 5, 3
    wide = (H + 2 * kv) * hd
    w = rng.integers(-127, 128, (wide, hidden)).astype(np.int8)
    ws = rng.uniform(1e-3, 2e-3, wide).astype(np.float32)
    wd, wsd = dev(torch, w), dev(torch, ws)
    cos, sin = P.tables(steps + 1, hd)
    c, s = dev(torch, cos), dev(torch, sin)
    rp = P4.rope(c, s, True)
    pages = seqs * width * 2
    tables = [np.arange(seqs * width).reshape(seqs, width), (seqs * width + np.arange(seqs * width)).reshape(seqs, width)]
    pool = P4.Pool(torch, pages, page, kv, hd, tables[0])
    xq, xs = torch.zeros(seqs, hidden, dtype=torch.int8, device="cuda"), torch.zeros(seqs, device="cuda")
    qkv = torch.zeros(seqs, wide, device="cuda")
    out = torch.zeros(seqs, H * hd, device="cuda")
    lens = np.zeros(seqs, np.int64)
    rows = [[[] for _ in range(kv)] for _ in range(seqs)]  # (K, V, mass) of each kv head
    st = P4.stream_of(torch)
    evictions = 0
    for step in range(steps):
        x = rng.normal(size=(seqs, hidden)).astype(np.float32)
        xd = dev(torch, x)
        _capi.check(lib.jyc_quantize_rows_i8(xd.data_ptr(), hidden, seqs, hidden, xq.data_ptr(), hidden, xs.data_ptr(), st))
        _capi.check(lib.jyc_matmul_i8(xq.data_ptr(), hidden, xs.data_ptr(), wd.data_ptr(), hidden, wsd.data_ptr(), None,
                                      qkv.data_ptr(), wide, seqs, wide, hidden, st))
        turn, pos = _ints(torch, np.full(seqs, step)), _ints(torch, lens)
        raw = host(qkv).astype(np.float64).reshape(seqs, -1, hd)
        # queries turned in place by their own call, keys as they are appended
        _capi.check(lib.jyc_rope_rows(qkv.data_ptr(), wide, qkv.data_ptr(), wide, seqs, H, hd, turn.data_ptr(), P4.ref(rp), st))
        seq = _ints(torch, np.arange(seqs))
        kp = qkv.data_ptr() + 4 * H * hd
        _capi.check(P4.append(torch, pool, kp, kp + 4 * kv * hd, wide, seqs, seq, pos, rp, turn))
        lens += 1
        lensd = _ints(torch, lens)
        mass0 = [pool.masses(b, lens[b], tables[0]).astype(np.float64) for b in range(seqs)]
        _capi.check(P4.attend(torch, pool, qkv, out, H, lensd))
        (kq, kst, klo), (vq, vst, vlo) = (P4.quantise(t) for t in (
            P4.turn(raw[:, H: H + kv], np.full(seqs, step), cos, sin, True), raw[:, H + kv:]))
        kval, vval = P4.values(kq, kst, klo), P4.values(vq, vst, vlo)
        for b in range(seqs):
            for h in range(kv):
                rows[b][h].append((kval[b, h], vval[b, h]))
        got = pool.rows(0, lens[0])
        for h in range(kv):
            assert np.array_equal(P4.values(got[0], got[1], got[2])[:, h], np.array([r[0] for r in rows[0][h]]))
            assert np.array_equal(P4.values(got[3], got[4], got[5])[:, h], np.array([r[1] for r in rows[0][h]]))
        _check(torch, rng, pool, qkv, out, mass0, H, lens)
        if lens.max() > 32:
            evictions += 1
            masses = [pool.masses(b, lens[b]) for b in range(seqs)]
            new_lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")
            kept = torch.zeros(seqs, kv, budget, dtype=torch.int32, device="cuda")
            _capi.check(P4.evict(torch, pool, lensd, budget, recent, _ints(torch, tables[1][:, :new_width]), new_lens, kept))
            for b in range(seqs):
                for h in range(kv):
                    keep = P4.kept_rows(masses[b][:, h], lens[b], budget, recent)
                    assert np.array_equal(host(kept)[b, h], keep)
                    rows[b][h] = [rows[b][h][i] for i in keep]
            tables.reverse()
            pool.table_host = np.ascontiguousarray(tables[0], np.int32)
            pool.table = dev(torch, pool.table_host)
            lens = host(new_lens).astype(np.int64)
    assert evictions == 1 and np.all(lens == budget + steps - 33)


def test_a_captured_step_replays_for_new_rows(cuda):
    """Products, rotation, append, attention and eviction captured as one graph, without a workspace, give on every replay
    the bits that the calls give."""
    torch = cuda
    rng = np.random.default_rng(31)
    lib = _capi.load()
    seqs, hidden, H, kv, hd, page, budget, width = 3, 96, 8, 2, 64, 16, 70, 12
    wide = (H + 2 * kv) * hd
    wd = dev(torch, rng.integers(-127, 128, (wide, hidden)).astype(np.int8))
    wsd = dev(torch, rng.uniform(1e-3, 2e-3, wide).astype(np.float32))
    cos, sin = P.tables(400, hd)
    c, s = dev(torch, cos), dev(torch, sin)
    rp = P4.rope(c, s, False)
    new_width = -(-budget // page)
    pages, both = _table(rng, seqs, width + new_width)
    newd = _ints(torch, both[:, width:])
    x, turn = torch.zeros(seqs, hidden, device="cuda"), _ints(torch, np.zeros(seqs))
    pos, lens = _ints(torch, np.zeros(seqs)), _ints(torch, np.ones(seqs))

    class Side:
        def __init__(self):
            self.pool = P4.Pool(torch, pages, page, kv, hd, both[:, :width])
            self.xq = torch.zeros(seqs, hidden, dtype=torch.int8, device="cuda")
            self.xs, self.qkv = torch.zeros(seqs, device="cuda"), torch.zeros(seqs, wide, device="cuda")
            self.out = torch.zeros(seqs, H * hd, device="cuda")
            self.nl = torch.zeros(seqs, dtype=torch.int32, device="cuda")
            self.kept = torch.zeros(seqs, kv, budget, dtype=torch.int32, device="cuda")

        def step(self):
            st, qkv = P4.stream_of(torch), self.qkv.data_ptr()
            _capi.check(lib.jyc_quantize_rows_i8(x.data_ptr(), hidden, seqs, hidden, self.xq.data_ptr(), hidden,
                                                 self.xs.data_ptr(), st))
            _capi.check(lib.jyc_matmul_i8(self.xq.data_ptr(), hidden, self.xs.data_ptr(), wd.data_ptr(), hidden,
                                          wsd.data_ptr(), None, qkv, wide, seqs, wide, hidden, st))
            _capi.check(lib.jyc_rope_rows(qkv, wide, qkv, wide, seqs, H + kv, hd, turn.data_ptr(), P4.ref(rp), st))
            k = qkv + 4 * H * hd
            _capi.check(P4.append(torch, self.pool, k, k + 4 * kv * hd, wide, seqs, None, pos))
            _capi.check(P4.attend(torch, self.pool, self.qkv, self.out, H, lens))
            _capi.check(P4.evict(torch, self.pool, lens, budget, 8, newd, self.nl, self.kept))

        def state(self):
            p = self.pool
            return [host(t).copy() for t in (self.qkv, self.out, self.nl, self.kept, p.k, p.v, p.kp, p.vp, p.mass)]

    once, again = Side(), Side()
    state = rng.integers(0, 1000)
    for side in (once, again):
        side.pool.put_random(np.random.default_rng(state), None)
        side.pool.mass.copy_(torch.from_numpy(np.random.default_rng(state).random(tuple(side.pool.mass.shape)).astype(np.float32)))
        side.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again.step()
    for n in ([192, 1, 70], [5, 71, 150], [100, 100, 100]):
        x.normal_()
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        pos.copy_(lens - 1)
        turn.copy_(lens + 200)
        once.step()
        graph.replay()
        for got, want in zip(again.state(), once.state()):
            assert np.array_equal(got, want)
        assert list(host(again.nl)) == [min(m, budget) for m in n]


def test_appends_and_evictions_on_two_streams(cuda):
    """Calls on two streams, of other sequences of one cache, give what they give one after another."""
    torch = cuda
    rng = np.random.default_rng(32)
    kv, hd, page, n, budget = 2, 64, 64, 6000, 500
    width, new_width = -(-n // page), -(-budget // page)
    pages, both = _table(rng, 2, width + new_width)
    K, V = (torch.randn(n, kv * hd, device="cuda") for _ in range(2))
    pos = _ints(torch, np.arange(n))
    weight = torch.from_numpy(rng.random((pages, page, kv)).astype(np.float32)).cuda()
    results = []
    for overlap in (False, True):
        pools = [P4.Pool(torch, pages, page, kv, hd, both[b: b + 1, :width]) for b in range(2)]
        shared = pools[0]
        for name in ("k", "v", "kp", "vp", "mass"):
            setattr(pools[1], name, getattr(shared, name))
        pools[1].desc = shared.desc
        streams = [torch.cuda.Stream() for _ in range(2)]
        seq, lens = _ints(torch, np.zeros(n)), _ints(torch, [n])
        nl, kept = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.zeros(2, 1, kv, budget, dtype=torch.int32, device="cuda")
        news = [_ints(torch, both[b: b + 1, width:]) for b in range(2)]
        torch.cuda.synchronize()
        for b, st in enumerate(streams):
            _capi.check(P4.append(torch, pools[b], K.data_ptr(), V.data_ptr(), kv * hd, n, seq, pos, stream=st.cuda_stream))
            if not overlap:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        shared.mass.copy_(weight)
        torch.cuda.synchronize()
        for b, st in enumerate(streams):
            _capi.check(P4.evict(torch, pools[b], lens, budget, 20, news[b], nl[b], kept[b], stream=st.cuda_stream))
            if not overlap:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        results.append([host(t).copy() for t in (shared.k, shared.v, shared.kp, shared.vp, shared.mass, nl, kept)])
    for a, b in zip(*results):
        assert np.array_equal(a, b)
    w = host(weight)
    for b in range(2):
        m = w[both[b, np.arange(n) // page], np.arange(n) % page]
        for h in range(kv):
            assert np.array_equal(results[0][-1][b, 0, h], P4.kept_rows(m[:, h], n, budget, 20))


def test_tables_without_room(cuda):
    """table_stride 0: no sequence has a place, empty ones give zeros and keep nothing."""
    torch = cuda
    lib = _capi.load()
    pool = P4.Pool(torch, 1, 16, 2, 64, np.zeros((2, 1)), fill=5)
    pool.table = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    some = torch.zeros(4, dtype=torch.int32, device="cuda")
    mass = pool.mass
    q, out = torch.randn(2, 4 * 64, device="cuda"), torch.full((2, 4 * 64), 3.0, device="cuda")
    for lens, bits in (([0, 0], 0), ([1, 0], 1)):
        n = _ints(torch, lens)
        _capi.check(lib.jyc_attention_paged_q4(q.data_ptr(), 256, out.data_ptr(), 256, 4, 2, 64, n.data_ptr(), some.data_ptr(),
                                               0, 2, None, None, P4.ref(pool.desc), None, 0, P4.stream_of(torch)))
        assert not host(out).any() and lib.jyc_paged_error(1) == bits
        out.fill_(3.0)
    x = torch.randn(2, 128, device="cuda")
    _capi.check(lib.jyc_kv_append_paged_q4(x.data_ptr(), x.data_ptr(), 128, 2, 2, 64, None, some.data_ptr(), some.data_ptr(), 0,
                                           2, None, None, P4.ref(pool.desc), P4.stream_of(torch)))
    assert lib.jyc_paged_error(1) == 1
    assert np.all(host(pool.k) == 5) and np.all(host(mass) == 5.0)
    kept, nl = (torch.full(s, 9, dtype=torch.int32, device="cuda") for s in ((2, 2, 8), (2,)))
    _capi.check(lib.jyc_kv_evict_paged_q4(_ints(torch, [0, 0]).data_ptr(), 8, 2, 2, 64, some.data_ptr(), 0, 2, some.data_ptr(), 1,
                                          nl.data_ptr(), kept.data_ptr(), P4.ref(pool.desc), P4.stream_of(torch)))
    assert np.all(host(kept) == -1) and np.all(host(nl) == 0)
