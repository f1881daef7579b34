"""jyc_sample_batch against the 64-bit definition of _paged.picks: the same token in every row,
except where a sum lies within the fixed-point rounding of a border (then either neighbour)."""
import numpy as np
import pytest

import _paged as P
from _util import dev, host
from jieyu_b200 import _capi

pytestmark = pytest.mark.gpu


def _call(torch, logits, V, T, k, p, mp, u, ids, probs, ld=None, stream=None):
    return _capi.load().jyc_sample_batch(
        logits.data_ptr(), logits.stride(0) if ld is None else ld, len(u), V, P.ptr(T), P.ptr(k), P.ptr(p), P.ptr(mp),
        P.ptr(u), P.ptr(ids), P.ptr(probs), torch.cuda.current_stream().cuda_stream if stream is None else stream)


def _run(torch, l, T=None, k=None, p=None, mp=None, u=None, pad=0, off=0):
    """l [rows][V] float32; returns ids and probabilities, and checks both against the definition."""
    rows, V = l.shape
    buf = np.full(rows * (V + pad) + off, 1e30, np.float32)  # what lies behind a row must not be read as logits
    buf[off:].reshape(rows, V + pad)[:, :V] = l
    d = dev(torch, buf)
    before = d.clone()
    asd = lambda x, t: None if x is None else dev(torch, np.asarray(x, t))  # noqa: E731
    Td, kd, pd, md, ud = asd(T, np.float32), asd(k, np.int32), asd(p, np.float32), asd(mp, np.float32), asd(u, np.float32)
    ids = torch.full((rows + 1,), -9, dtype=torch.int32, device="cuda")
    probs = torch.full((rows + 1,), -9.0, device="cuda")
    view = d[off:].as_strided((rows, V), (V + pad, 1))
    _capi.check(_call(torch, view, V, Td, kd, pd, md, ud, ids, probs, ld=V + pad))
    gi, gp = host(ids), host(probs)
    assert gi[rows] == -9 and gp[rows] == -9.0
    assert np.array_equal(host(d).view(np.uint32), host(before).view(np.uint32))
    at = lambda x, r, t: None if x is None else t(x[r])  # noqa: E731
    for r in range(rows):
        want = P.picks(l[r], 1.0 if T is None else np.float32(T[r]), at(k, r, int), at(p, r, float), at(mp, r, float),
                       u[r])
        assert int(gi[r]) in want, (r, int(gi[r]), want)
        # the quotient of two sums that each carry the fixed-point rounding, rounded to fp32 (and
        # 2^-40 for a border token moved in or out of the sum when several picks are allowed)
        tol = want[int(gi[r])] * (P.U24 + V * 2.0 ** -42 + 2.0 ** -43) + 2.0 ** -42
        if len(want) == 1:
            assert abs(gp[r] - want[int(gi[r])]) <= tol, (r, gp[r], want)
    again = torch.empty_like(ids)
    _capi.check(_call(torch, view, V, Td, kd, pd, md, ud, again, None, ld=V + pad))
    assert np.array_equal(host(again)[:rows], gi[:rows])
    return gi[:rows], gp[:rows]


def _logits(rng, rows, V, kind):
    l = (2.5 * rng.normal(size=(rows, V))).astype(np.float32)
    for r in range(rows):
        n = min(V, 24)
        l[r, rng.choice(V, n, replace=False)] = (8 + 6 * rng.random(n)).astype(np.float32)
    if kind == "bf16":  # many equal logits
        l = (l.view(np.uint32) & 0xFFFF0000).view(np.float32)
    elif kind == "equal":
        l[:] = 3.25
    elif kind == "two":
        l = np.where(rng.random((rows, V)) < 0.3, np.float32(2.0), np.float32(1.0)).astype(np.float32)
    elif kind == "masked":
        l[rng.random((rows, V)) < 0.9] = -np.inf
        l[rng.random((rows, V)) < 0.02] = np.nan
        l[:, V // 2] = 1.0
    elif kind == "lowest":  # a mask of the type's lowest value
        l[rng.random((rows, V)) < 0.9] = np.finfo(np.float32).min
        l[:, V // 2] = 1.0
    elif kind == "huge":
        l = (l * 1e37).astype(np.float32)
    elif kind == "tiny":
        l = (l * 1e-39).astype(np.float32)
    elif kind == "falling":
        l = -np.sort(-l, axis=1)
    elif kind == "flat":
        l = (l * 0.01).astype(np.float32)
    elif kind == "peak":
        l[:, V // 3] = 60.0
    return l


SETTINGS = [  # temperature, top-k, top-p, min-p
    (None, None, None, None), (0.7, 50, None, None), (1.0, None, 0.9, None), (1.3, None, None, 0.05),
    (0.8, 40, 0.95, 0.02), (1.0, 1, 0.5, None), (2.0, 3000, 0.999, None), (0.05, 10, 0.3, 0.5),
    (1.0, 0, 1.0, 0.0), (5.0, None, 0.5, None), (1.0, None, 0.0, None), (1.0, 2, 1.5, -1.0),
]


@pytest.mark.parametrize("V", [1, 2, 17, 1000, 1023, 4097, 32000])
@pytest.mark.parametrize("kind", ["plain", "bf16", "equal", "two", "masked", "lowest", "huge", "tiny", "falling",
                                  "flat", "peak"])
def test_picks(cuda, V, kind):
    rng = np.random.default_rng(V * 13 + len(kind))
    l = _logits(rng, len(SETTINGS), V, kind)
    u = rng.random(len(SETTINGS)).astype(np.float32)
    for i in range(3):
        off = {0: 1.0, 1: 0, 2: 1.0, 3: 0.0}
        col = lambda c: [s[c] if s[c] is not None else off[c] for s in SETTINGS]  # noqa: E731
        _run(cuda, l, col(0), col(1), col(2), col(3), u, pad=(0, 3, 4)[i], off=(0, 1, 0)[i])
        u = rng.random(len(SETTINGS)).astype(np.float32)


@pytest.mark.parametrize("T,k,p,mp", SETTINGS)
def test_arrays_may_be_absent(cuda, T, k, p, mp):
    rng = np.random.default_rng(77)
    rows = 5
    l = _logits(rng, rows, 5003, "plain")
    full = lambda x: None if x is None else [x] * rows  # noqa: E731
    _run(cuda, l, full(T), full(k), full(p), full(mp), rng.random(rows).astype(np.float32))


@pytest.mark.parametrize("rows,V", [(1, 151936), (3, 128256), (40, 50257), (300, 2048), (700, 3), (1, 1 << 20)])
def test_large(cuda, rows, V):
    rng = np.random.default_rng(V)
    l = _logits(rng, rows, V, "plain")
    i = np.arange(rows) if rows > 1 else np.array([4])
    _run(cuda, l, np.where(i % 5 == 0, 0.0, 0.5 + rng.random(rows)), np.where(i % 3 == 1, 50, 0),
         np.where(i % 2 == 0, 0.9, 1.0), np.where(i % 7 == 2, 0.05, 0.0), rng.random(rows).astype(np.float32))


def test_large_k_and_hot_rows(cuda):
    """k around the largest that a CTA's maxima bound (2048) and beyond it, temperatures that leave one
    token or all of them, and top-p next to 1."""
    rng = np.random.default_rng(11)
    V = 50000
    k = [1023, 1024, 1025, 2047, 2048, 2049, 4000, 49999, 0, 0, 0, 0, 0, 3000, 2048, 700]
    n = len(k)
    l = _logits(rng, n, V, "plain")
    T = [1.0, 0.7, 1.3, 1.0, 2.0, 1.0, 1.0, 1.0, 1e-38, 1e-30, 1e4, 30.0, 1.3, 1.0, 5.0, 1e30]
    p = [1.0, 0.9, 1.0, 0.99, 1.0, 0.5, 0.95, 0.9, 0.9, 1.0, 0.7, 0.99, 1 - 2.0 ** -24, 1 - 2.0 ** -23, 0.9, 0.3]
    for mp in (0.0, 1e-4):
        _run(cuda, l, T, k, p, [mp] * n, rng.random(n).astype(np.float32))


@pytest.mark.parametrize("kind", ["flat", "equal", "bf16", "two"])
def test_large_and_flat(cuda, kind):
    """Borders that fall among tens of thousands of (nearly) equal logits."""
    rng = np.random.default_rng(5)
    rows, V = 6, 128256
    l = _logits(rng, rows, V, kind)
    _run(cuda, l, [1.0] * rows, [0, 60000, 0, 100000, 1, 0], [0.5, 1.0, 0.9, 0.7, 0.5, 1.0], [0, 0, 0, 0, 0, 0.9],
         rng.random(rows).astype(np.float32))


def test_border_among_logits_of_both_signs(cuda):
    """The border's tokens lie in one narrow bin, on both sides of zero and over ten decades."""
    rng = np.random.default_rng(19)
    high, low = 2100, 400
    k = [0, 0, 0, 2150, 2300, 2301, 2499, 2300]
    n = len(k)
    l = np.empty((n, high + low), np.float32)
    for r in range(n):
        x = np.concatenate([5e9 * (1 - 1e-3 * rng.random(high)),
                            rng.choice([-1, 1], low) * 10.0 ** rng.uniform(-5, 5, low)])
        l[r] = rng.permutation(x)
    w = np.exp((l[0].astype(np.float64) - l[0].max()) / 1e9)
    tail = w[l[0] < 1e9].sum() / w.sum()
    p = [1 - 0.5 * tail, 1 - 0.9 * tail, 1 - 0.01 * tail, 1.0, 1.0, 1.0, 1.0, 1 - 0.3 * tail]
    for u in (rng.random(n), 1 - 0.5 * tail * rng.random(n)):
        _run(cuda, l, [1e9] * n, k, p, None, np.minimum(u, 1 - 2.0 ** -24).astype(np.float32))


def test_draws_at_the_ends(cuda):
    """u of 0, just below 1, and out of range or NaN: always a kept token."""
    l = np.full((6, 50), -np.inf, np.float32)
    l[:, [7, 20, 33]] = [0.0, 1.0, 0.5]
    u = np.array([0.0, 1 - 2.0 ** -24, 1.0, 2.0, -0.5, np.nan], np.float32)
    torch = cuda
    d, ud = dev(torch, l), dev(torch, u)
    ids = torch.empty(6, dtype=torch.int32, device="cuda")
    _capi.check(_call(torch, d, 50, None, None, None, None, ud, ids, None))
    assert host(ids).tolist() == [7, 33, 33, 33, 7, 33]


def test_greedy_rows_equal_argmax(cuda):
    torch = cuda
    rng = np.random.default_rng(2)
    V = 5000
    l = np.round(3 * rng.normal(size=(4, V))).astype(np.float32)  # ties everywhere
    l[1, 17] = np.nan
    l[2, :] = -0.0
    l[2, 5] = 0.0
    d = dev(torch, l)
    ids = torch.empty(4, dtype=torch.int32, device="cuda")
    probs = torch.empty(4, device="cuda")
    T = dev(torch, np.array([0.0, -1.0, np.nan, 0.0], np.float32))
    u = dev(torch, np.zeros(4, np.float32))
    _capi.check(_call(torch, d, V, T, None, None, None, u, ids, probs))
    got = host(ids)
    for r in (0, 1, 3):
        one = torch.empty(1, dtype=torch.int32, device="cuda")
        _capi.check(_capi.load().jyc_argmax(d[r].data_ptr(), V, one.data_ptr(), torch.cuda.current_stream().cuda_stream))
        assert got[r] == int(one)
    assert got[2] == 0  # the two zeros are equal
    assert np.all(host(probs) == 1.0)


def test_rows_that_hold_nothing_and_infinities(cuda):
    torch = cuda
    V = 300
    l = np.zeros((6, V), np.float32)
    l[0] = -np.inf
    l[1] = np.nan
    l[2, ::2], l[2, 1::2] = np.nan, -np.inf
    l[3, [10, 200]] = np.inf
    l[4] = -np.inf
    l[4, 99] = -3e38
    l[5, 250] = np.inf
    for T in (0.0, 1.0, np.inf):
        T6 = np.full(6, T, np.float32)
        d = dev(torch, l)
        ids = torch.empty(6, dtype=torch.int32, device="cuda")
        probs = torch.empty(6, device="cuda")
        u = dev(torch, np.full(6, 0.75, np.float32))
        _capi.check(_call(torch, d, V, dev(torch, T6), None, None, None, u, ids, probs))
        got, p = host(ids), host(probs)
        assert got[:3].tolist() == [-1, -1, -1] and np.all(p[:3] == 0.0)
        assert got[3] == (10 if T == 0 else 200) and p[3] == (1.0 if T == 0 else 0.5)
        assert got[4] == 99 and p[4] == 1.0
        assert got[5] == 250 and p[5] == 1.0


def test_captured_and_on_two_streams(cuda):
    torch = cuda
    rng = np.random.default_rng(6)
    rows, V = 9, 20000
    l = [_logits(rng, rows, V, "plain") for _ in range(3)]
    k = dev(torch, np.full(rows, 30, np.int32))
    d = dev(torch, l[0])
    u = rng.random(rows).astype(np.float32)
    ud = dev(torch, u)
    ids = torch.empty(rows, dtype=torch.int32, device="cuda")
    _capi.check(_call(torch, d, V, None, k, None, None, ud, ids, None))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _capi.check(_call(torch, d, V, None, k, None, None, ud, ids, None))
    for x in l:
        d.copy_(torch.from_numpy(x))
        g.replay()
        got = host(ids)
        assert all(int(got[r]) in P.picks(x[r], 1.0, 30, None, None, u[r]) for r in range(rows))
    streams = [torch.cuda.Stream() for _ in range(2)]
    ds = [dev(torch, x) for x in l[:2]]
    outs = [torch.empty(rows, dtype=torch.int32, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            _capi.check(_call(torch, ds[i], V, None, k, None, None, ud, outs[i], None, stream=streams[i].cuda_stream))
    torch.cuda.synchronize()
    for i in range(2):
        got = host(outs[i])
        assert all(int(got[r]) in P.picks(l[i][r], 1.0, 30, None, None, u[r]) for r in range(rows))


def test_distribution(cuda):
    """Equally spaced u sweep the inverse CDF: each token is picked as often as its weight says, to one."""
    torch = cuda
    rng = np.random.default_rng(4)
    V, n = 40, 4096
    row = rng.normal(size=V).astype(np.float32)
    l = np.repeat(row[None], n, 0)
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    ids, probs = _run(torch, l, [1.1] * n, [20] * n, [0.9] * n, [0.0] * n, u)
    keep = np.unique(ids)
    w = P.weights(row, np.float64(np.float32(1.1)))[1][keep]
    count = np.array([(ids == i).sum() for i in keep])
    assert np.all(np.abs(count - n * w / w.sum()) <= 1.0 + 1e-6)
    assert np.all(np.diff(ids) >= 0)


@pytest.mark.parametrize("rows,V", [(1, 65536), (60, 65536), (150, 32768), (37, 131072)])
def test_clusters_that_start_late(cuda, rows, V):
    """Rows of 2 to 8 CTAs while another stream's kernels hold most of the SMs, so that the CTAs of a row
    find their places at different times: every call gives the picks of the definition."""
    torch = cuda
    rng = np.random.default_rng(rows + V)
    l = _logits(rng, rows, V, "plain")
    u = rng.random(rows).astype(np.float32)
    d, ud = dev(torch, l), dev(torch, u)
    k = dev(torch, np.full(rows, 40, np.int32))
    want = [P.picks(l[r], 1.0, 40, None, None, u[r]) for r in range(rows)]
    ids = torch.full((32, rows), -9, dtype=torch.int32, device="cuda")
    busy, here = torch.cuda.Stream(), torch.cuda.Stream()
    a = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for i in range(32):
        with torch.cuda.stream(busy):
            a.mul_(1.0).add_(0.0)
        _capi.check(_call(torch, d, V, None, k, None, None, ud, ids[i], None, stream=here.cuda_stream))
    torch.cuda.synchronize()
    got = host(ids)
    for r in range(rows):
        assert set(got[:, r].tolist()) <= set(want[r]), r


@pytest.mark.parametrize("V", [4000, 10001, 70000])
def test_k_above_the_number_of_tokens(cuda, V):
    """A large k over a row with fewer logits than that (the others -inf or NaN), more than a thousand of
    which lie far below the maximum, down to the type's lowest value: all of them are kept."""
    rng = np.random.default_rng(V)
    k = [0.6, 0.5, 0.45, 0.9, 0.41, 0.399]  # of V; 0.4 of V are logits
    rows, n = len(k), 2 * V // 5
    l = np.full((rows, V), -np.inf, np.float32)
    for r in range(rows):
        at = rng.permutation(V)
        x = np.concatenate([[0.0], np.full(3 * n // 4, -40.0), -(10.0 ** rng.uniform(np.log10(40), 38, n))])[:n]
        x[n // 2] = np.finfo(np.float32).min
        if r % 2:
            x[1: n // 4] = -rng.random(n // 4 - 1)  # some with weight
        l[r, at[:n]] = x
        l[r, at[n: n + V // 5]] = np.nan
    k = [int(f * V) for f in k]
    for u in (rng.random(rows), np.full(rows, 1 - 2.0 ** -24)):
        _run(cuda, l, [1.0] * rows, k, None, [0.0, 0.0, 0.5, 0.5, 0.0, 0.0], u.astype(np.float32))


def _group_borders(rng, x, T, rows):
    """top-p values whose border falls around the end of a group of equal logits of x."""
    values, count = np.unique(x, return_counts=True)
    w = P.weights(values, np.float64(np.float32(T)))[1]
    upto = np.cumsum((count * w)[::-1])
    at = rng.integers(0, len(values), rows)
    off = np.array([0.5, 0.02, 0.98, -0.5, 1.5, 0.3])[np.arange(rows) % 6]  # of the group's last token
    return np.clip((upto[at] - off * w[::-1][at]) / upto[-1], 1e-6, 1 - 2.0 ** -24)


@pytest.mark.parametrize("V", [5000, 20000, 131072])
@pytest.mark.parametrize("kind", ["two", "near", "steps", "bf16", "equal"])
def test_borders_at_the_end_of_equal_logits(cuda, V, kind):
    """Thousands of equal logits beside others that weigh almost the same, the border of top-p in the last
    token of a group or beside it; with a large top-k too."""
    rng = np.random.default_rng(V + len(kind))
    rows = 12
    l = np.empty((rows, V), np.float32)
    T = [1.0, 0.7, 1.0, 3.0] * 3
    for r in range(rows):
        if kind == "two":
            l[r] = np.where(rng.permutation(V) < V // 2, 1.0, 0.99)
        elif kind == "near":
            l[r] = np.where(rng.permutation(V) < V - 1 - r, 4.0, 3.984375)
        elif kind == "steps":
            l[r] = rng.choice([4.0, 3.984375, 3.96875, 2.0], V)
        elif kind == "bf16":
            l[r] = ((4 + 0.02 * rng.normal(size=V)).astype(np.float32).view(np.uint32) & 0xFFFF0000).view(np.float32)
        else:
            l[r] = 3.25
    p = [_group_borders(rng, l[r], T[r], rows)[r] for r in range(rows)]
    k = np.where(np.arange(rows) % 4 == 3, V - 7, 0)
    for u in (rng.random(rows), np.full(rows, 1 - 2.0 ** -24)):
        _run(cuda, l, T, k, p, None, u.astype(np.float32))


def _allowed(l, T, k, p, mp, u):
    """Every (id, probability) that the definition allows: where the border of top-p lies within the rounding
    of the sums (with equal weights it may lie on one exactly), one token more or fewer is kept, and the same
    id comes with either probability. A prefix by top-p is a prefix by count."""
    l64, w = P.weights(l, np.float64(np.float32(T)))
    order = np.argsort(-l64, kind="stable")[: k if 0 < k < len(l) else len(l)]
    ns = {len(order)}
    if p < 1:
        sums, slack = np.cumsum(w[order]), len(l) * 2.0 ** -43 + 2.0 ** -44 * w.sum()
        need = np.float64(np.float32(p)) * sums[-1]
        ns = {1 + int(np.searchsorted(sums, x)) for x in (need, need - slack, need + slack)}
    return {x for n in ns for x in P.picks(l, T, max(1, n), None, mp, u).items()}


def _run_at_borders(torch, l, T, k, p, mp, u):
    rows, V = l.shape
    d, ud = dev(torch, l), dev(torch, u)
    args = [dev(torch, np.asarray(x, t)) for x, t in ((T, np.float32), (k, np.int32), (p, np.float32), (mp, np.float32))]
    ids = torch.full((rows,), -9, dtype=torch.int32, device="cuda")
    probs = torch.full((rows,), -9.0, device="cuda")
    _capi.check(_call(torch, d, V, *args, ud, ids, probs))
    gi, gp = host(ids), host(probs)
    for r in range(rows):
        want = _allowed(l[r], T[r], k[r], p[r], mp[r], u[r])
        assert any(i == gi[r] and abs(gp[r] - q) <= q * (P.U24 + V * 2.0 ** -42 + 2.0 ** -43) + 2.0 ** -42
                   for i, q in want), (r, gi[r], gp[r], want)


@pytest.mark.parametrize("V", [2, 300, 6000, 40000])
@pytest.mark.parametrize("T", [1e38, 3e37, 3e38, np.inf])
def test_logits_over_the_whole_range(cuda, V, T):
    """Logits of both signs next to the type's limits, whose differences fp32 does not hold, at temperatures
    that leave them weight: top-p, min-p, top-k and all of them."""
    rng = np.random.default_rng(V)
    settings = [(0, 1.0, 0.0), (0, 1.0, 1e-3), (0, 1.0, 0.05), (0, 0.999, 0.0), (0, 0.9, 0.0), (0, 0.5, 0.01),
                (V // 2, 1.0, 0.0), (V // 2, 0.7, 0.0), (3, 0.9, 0.0), (0, 1 - 2.0 ** -20, 0.0)]
    rows = len(settings)
    l = (3.4e38 * rng.uniform(-1, 1, (rows, V))).astype(np.float32)
    l[:, 0], l[:, -1] = 3e38, -3e38
    l[1::3, V // 3] = np.finfo(np.float32).min
    l[2::3, V // 2] = np.finfo(np.float32).max
    if V > 2:
        l[:, 1], l[:, 2] = np.nan, -np.inf
    k, p, mp = zip(*settings)
    for u in (rng.random(rows), np.full(rows, 1 - 2.0 ** -24), np.zeros(rows)):
        _run_at_borders(cuda, l, [T] * rows, k, p, mp, u.astype(np.float32))


@pytest.mark.parametrize("T", [1e-30, 7e-29, 3e-38, 1.5e-44])
def test_tiny_temperatures(cuda, T):
    """Thousands of tokens with weight at temperatures near the least that fp32 holds: logits of T's own
    size, around zero or all of one sign, and beside them ordinary ones."""
    rng = np.random.default_rng(3)
    V = 20000
    settings = [(0, 0.5, 0.0), (0, 0.9, 0.0), (0, 0.999, 0.0), (0, 1.0, 0.01), (5000, 0.7, 0.0), (40, 0.9, 0.0),
                (0, 1 - 2.0 ** -20, 0.0), (0, 1.0, 0.0), (0, 0.8, 0.05)]
    rows = len(settings)
    T = float(np.float32(T))
    l = np.empty((rows, V), np.float32)
    for r in range(rows):
        l[r] = (T * (rng.choice([-40.0, 0.0, 25.0]) + 20 * rng.random(V))).astype(np.float32)
        l[r, rng.integers(0, V, 50)] = -1.0
        l[r, rng.integers(0, V, 50)] = -np.inf
    k, p, mp = zip(*settings)
    for u in (rng.random(rows), np.full(rows, 1 - 2.0 ** -24)):
        _run_at_borders(cuda, l, [T] * rows, k, p, mp, u.astype(np.float32))


def test_nan_filters_are_off(cuda):
    """NaN in top-p or min-p means the filter's default, as for a row without it."""
    torch = cuda
    rng = np.random.default_rng(8)
    rows, V = 40, 900
    l = _logits(rng, 1, V, "plain").repeat(rows, 0)
    u = ((np.arange(rows) + 0.5) / rows).astype(np.float32)
    d, ud = dev(torch, l), dev(torch, u)
    nan, k = dev(torch, np.full(rows, np.nan, np.float32)), dev(torch, np.full(rows, 200, np.int32))
    got = []
    for p, mp in ((None, None), (nan, None), (None, nan), (nan, nan)):
        for top_k in (None, k):
            ids = torch.full((rows,), -9, dtype=torch.int32, device="cuda")
            probs = torch.zeros(rows, device="cuda")
            _capi.check(_call(torch, d, V, None, top_k, p, mp, ud, ids, probs))
            got.append((host(ids), host(probs)))
    for i in range(2, len(got)):
        assert np.array_equal(got[i][0], got[i % 2][0]) and np.array_equal(got[i][1], got[i % 2][1]), i
    assert len(set(got[0][0].tolist())) > 1
