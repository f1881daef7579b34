"""jyc_quantize_rows_i8 and jyc_matmul_i8 on the device. The whole-number sums are exact, so outputs
equal the defined roundings of the 64-bit result bit for bit."""
import numpy as np
import pytest

import _paged as P
from _util import dev, host
from jieyu_b200 import _capi

pytestmark = pytest.mark.gpu


def _stream(torch):
    return torch.cuda.current_stream().cuda_stream


def _expected(a, sa, w, sw, bias):
    """fp32(sum) * fp32(sa sw), + bias: one rounding each."""
    whole = a.astype(np.float64) @ w.astype(np.float64).T
    y = P.r32(P.r32(whole) * P.r32(sa.astype(np.float64)[:, None] * sw.astype(np.float64)))
    return (P.r32(y + bias.astype(np.float64)) if bias is not None else y).astype(np.float32)


def _run(torch, a, sa, w, sw, bias, m, n, k, pa=0, pw=0, pc=0, fill=77, offset=0):
    """Product of [m][k] and [n][k] with spare bytes behind the rows (of random content) and spare floats behind C's."""
    lda, ldw, ldc = -(-k // 16) * 16 + 16 * pa, -(-k // 16) * 16 + 16 * pw, n + pc
    rng = np.random.default_rng(1)
    ah, wh = rng.integers(-128, 128, (m, lda)).astype(np.int8), rng.integers(-128, 128, (n, ldw)).astype(np.int8)
    ah[:, :k], wh[:, :k] = a, w
    ad, wd, sad, swd = dev(torch, ah), dev(torch, wh), dev(torch, sa), dev(torch, sw)
    bd = None if bias is None else dev(torch, bias)
    c = torch.full((m * ldc + offset,), float(fill), device="cuda")
    _capi.check(_capi.load().jyc_matmul_i8(ad.data_ptr(), lda, sad.data_ptr(), wd.data_ptr(), ldw, swd.data_ptr(),
                                           P.ptr(bd), c.data_ptr() + 4 * offset, ldc, m, n, k, _stream(torch)))
    got = host(c)
    assert np.all(got[:offset] == fill)
    got = got[offset:].reshape(m, ldc)
    assert np.all(got[:, n:] == fill)
    return got[:, :n]


def _inputs(rng, m, n, k):
    return (rng.integers(-127, 128, (m, k)).astype(np.int8), rng.uniform(1e-4, 2e-3, m).astype(np.float32),
            rng.integers(-128, 128, (n, k)).astype(np.int8), rng.uniform(1e-4, 2e-3, n).astype(np.float32))


SHAPES = [(1, 1, 1), (1, 16, 16), (1, 128, 128), (1, 300, 1000), (2, 7, 31), (3, 129, 4090), (5, 64, 127), (8, 256, 512),
          (9, 130, 333), (16, 1000, 640), (17, 40, 2048), (31, 257, 96), (33, 512, 129), (48, 384, 4090),
          (64, 128, 1024), (65, 255, 257), (100, 500, 300), (127, 129, 130), (128, 256, 128), (129, 1024, 4096),
          (200, 127, 1000), (256, 256, 384), (257, 513, 700), (300, 2000, 64), (640, 384, 1111), (1000, 136, 272),
          # many tiles: one or several for each SM, ragged in every direction
          (520, 4160, 130), (1300, 4200, 200), (700, 13001, 64), (129, 19000, 417), (2049, 2500, 900)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(cuda, m, n, k):
    rng = np.random.default_rng(m * 31 + n * 7 + k)
    a, sa, w, sw = _inputs(rng, m, n, k)
    bias = rng.normal(size=n).astype(np.float32) if (m + n + k) % 2 else None
    got = _run(cuda, a, sa, w, sw, bias, m, n, k)
    assert np.array_equal(got, _expected(a, sa, w, sw, bias))


@pytest.mark.parametrize("m", [1, 6, 24, 70, 200])
@pytest.mark.parametrize("pa,pw,pc,offset", [(1, 0, 3, 1), (0, 5, 1, 2), (3, 3, 4, 4), (2, 1, 0, 3)])
def test_strides(cuda, m, pa, pw, pc, offset):
    rng = np.random.default_rng(m)
    n, k = 150, 417
    a, sa, w, sw = _inputs(rng, m, n, k)
    bias = rng.normal(size=n).astype(np.float32)
    assert np.array_equal(_run(cuda, a, sa, w, sw, bias, m, n, k, pa, pw, pc, offset=offset),
                          _expected(a, sa, w, sw, bias))


@pytest.mark.parametrize("m", [1, 12, 40, 150])
@pytest.mark.parametrize("va,vw", [(-128, -128), (127, -128), (127, 127)])
def test_largest_sums(cuda, m, va, vw):
    """k = 131071 of the largest products: the sums reach 2^31 - 2^14."""
    n, k = 20, 131071
    a, w = np.full((m, k), va, np.int8), np.full((n, k), vw, np.int8)
    sa, sw = np.linspace(0.5, 2, m).astype(np.float32), np.linspace(1e-3, 1, n).astype(np.float32)
    assert np.array_equal(_run(cuda, a, sa, w, sw, None, m, n, k), _expected(a, sa, w, sw, None))


@pytest.mark.parametrize("m", [2, 33, 140])
def test_scales_that_are_not_numbers(cuda, m):
    """An infinite row scale makes its row infinite or NaN, and no other."""
    rng = np.random.default_rng(4)
    n, k = 70, 200
    a, sa, w, sw = _inputs(rng, m, n, k)
    sa[1], sw[5], sw[6] = np.inf, np.nan, 0.0
    a[1] = 0
    with np.errstate(invalid="ignore"):
        want = _expected(a, sa, w, sw, None)
    got = _run(cuda, a, sa, w, sw, None, m, n, k)
    assert np.array_equal(got, want, equal_nan=True)
    assert np.isnan(got[1]).all() and np.isnan(got[:, 5]).all() and np.isfinite(got[0, :5]).all()


@pytest.mark.parametrize("rows,k,extra,off", [(1, 1, 0, 0), (3, 7, 5, 1), (2, 4096, 0, 0), (5, 4090, 2, 0),
                                              (70, 333, 1, 3), (2, 20000, 0, 0), (1, 14336, 4, 0), (300, 128, 0, 0),
                                              (2, 131071, 1, 0), (9, 8192, 0, 0), (9, 8196, 0, 0)])
def test_quantize_rows(cuda, rows, k, extra, off):
    torch = cuda
    rng = np.random.default_rng(rows + k)
    ldx, ldq = k + extra, -(-k // 16) * 16
    x = rng.normal(size=off + rows * ldx).astype(np.float32)
    body = x[off:].reshape(rows, ldx)
    body[:, k:] = 1e9  # behind the row: does not count
    if rows > 4:
        body[0, :k] = 0.0
        body[1, :k] *= np.float32(1e-12)
        body[2, k // 2] = np.nan
        body[3, k // 3] = -np.inf
        body[4, 0] = 3e38
    xd = dev(torch, x)
    q = torch.full((rows, ldq), 55, dtype=torch.int8, device="cuda")
    s = torch.zeros(rows, device="cuda")
    _capi.check(_capi.load().jyc_quantize_rows_i8(xd.data_ptr() + 4 * off, ldx, rows, k, q.data_ptr(), ldq,
                                                  s.data_ptr(), _stream(torch)))
    wq, ws = P.quantise(body[:, :k].astype(np.float64))
    got = host(q)
    assert np.array_equal(got[:, :k], wq.astype(np.int8)) and np.all(got[:, k:] == 55)
    assert np.array_equal(host(s), ws.astype(np.float32))


def test_whole_projection(cuda):
    """Activations through both calls stand near their fp32 product: each value is off by half a step of its scale."""
    torch = cuda
    rng = np.random.default_rng(8)
    m, n, k = 37, 200, 1000
    x, w = rng.normal(size=(m, k)).astype(np.float32), rng.normal(size=(n, k)).astype(np.float32)
    ldq = -(-k // 16) * 16
    xd, wd = dev(torch, x), dev(torch, w)
    qa, qw = (torch.zeros(r, ldq, dtype=torch.int8, device="cuda") for r in (m, n))
    sa, sw = torch.zeros(m, device="cuda"), torch.zeros(n, device="cuda")
    lib, st = _capi.load(), _stream(torch)
    _capi.check(lib.jyc_quantize_rows_i8(xd.data_ptr(), k, m, k, qa.data_ptr(), ldq, sa.data_ptr(), st))
    _capi.check(lib.jyc_quantize_rows_i8(wd.data_ptr(), k, n, k, qw.data_ptr(), ldq, sw.data_ptr(), st))
    c = torch.zeros(m, n, device="cuda")
    _capi.check(lib.jyc_matmul_i8(qa.data_ptr(), ldq, sa.data_ptr(), qw.data_ptr(), ldq, sw.data_ptr(), None,
                                  c.data_ptr(), n, m, n, k, st))
    x, w, sa, sw = x.astype(np.float64), w.astype(np.float64), host(sa).astype(np.float64), host(sw).astype(np.float64)
    # |x w - x' w'| <= |x| sw/2 + |w| sa/2 + sa sw/4 for each of k terms, and three roundings of the result
    bound = (np.abs(x).sum(-1)[:, None] * sw / 2 + sa[:, None] / 2 * np.abs(w).sum(-1) + k * sa[:, None] * sw / 4)
    want = x @ w.T
    assert np.all(np.abs(host(c) - want) <= bound * (1 + 1e-6) + 4 * P.U24 * np.abs(want))


def test_graph_replays(cuda):
    torch = cuda
    rng = np.random.default_rng(9)
    lib = _capi.load()
    for m in (4, 150):
        n, k = 260, 512
        a, sa, w, sw = _inputs(rng, m, n, k)
        ad, sad, wd, swd = dev(torch, a), dev(torch, sa), dev(torch, w), dev(torch, sw)
        c = torch.zeros(m, n, device="cuda")
        call = lambda s: lib.jyc_matmul_i8(ad.data_ptr(), k, sad.data_ptr(), wd.data_ptr(), k, swd.data_ptr(), None,  # noqa: E731
                                           c.data_ptr(), n, m, n, k, s)
        _capi.check(call(_stream(torch)))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _capi.check(call(torch.cuda.current_stream().cuda_stream))
        for _ in range(2):
            a = rng.integers(-127, 128, (m, k)).astype(np.int8)
            ad.copy_(torch.from_numpy(a))
            c.zero_()
            graph.replay()
            assert np.array_equal(host(c), _expected(a, sa, w, sw, None))


def test_two_streams(cuda):
    """Calls that overlap in time do not share anything."""
    torch = cuda
    rng = np.random.default_rng(10)
    lib = _capi.load()
    for m in (3, 40, 300):
        n, k = 700, 1024
        sets = []
        for _ in range(2):
            a, sa, w, sw = _inputs(rng, m, n, k)
            sets.append((a, sa, w, sw, [dev(torch, t) for t in (a, sa, w, sw)], torch.zeros(m, n, device="cuda"),
                         torch.cuda.Stream()))
        torch.cuda.synchronize()
        for _ in range(4):
            for a, sa, w, sw, (ad, sad, wd, swd), c, st in sets:
                _capi.check(lib.jyc_matmul_i8(ad.data_ptr(), k, sad.data_ptr(), wd.data_ptr(), k, swd.data_ptr(), None,
                                              c.data_ptr(), n, m, n, k, st.cuda_stream))
        for a, sa, w, sw, _, c, _ in sets:
            assert np.array_equal(host(c), _expected(a, sa, w, sw, None))


@pytest.mark.parametrize("va,vw", [(-128, -128), (127, -128), (None, None)])
def test_largest_sums_of_pairs_of_ctas(cuda, va, vw):
    """k = 131071 where there are tiles of 256 x 256 for a quarter of the SMs: the form whose CTAs work in pairs."""
    torch = cuda
    m, n, k, ld = 300, 4865, 131071, 131072
    if va is None:
        a, w = (torch.randint(-128, 128, (r, ld), dtype=torch.int8, device="cuda") for r in (m, n))
    else:
        a = torch.full((m, ld), va, dtype=torch.int8, device="cuda")
        w = torch.full((n, ld), vw, dtype=torch.int8, device="cuda")
    sa, sw = np.linspace(0.5, 2, m).astype(np.float32), np.linspace(1e-3, 1, n).astype(np.float32)
    bias = np.random.default_rng(3).normal(size=n).astype(np.float32)
    sad, swd, bd = dev(torch, sa), dev(torch, sw), dev(torch, bias)
    c = torch.full((m, n + 3), 7.0, device="cuda")
    _capi.check(_capi.load().jyc_matmul_i8(a.data_ptr(), ld, sad.data_ptr(), w.data_ptr(), ld, swd.data_ptr(), bd.data_ptr(),
                                           c.data_ptr(), n + 3, m, n, k, _stream(torch)))
    if va is None:
        whole = torch.cat([a[:, :k].double() @ w[j: j + 500, :k].double().T for j in range(0, n, 500)], 1).cpu().numpy()
    else:
        whole = np.full((m, n), float(va) * vw * k)
    y = P.r32(P.r32(whole) * P.r32(sa.astype(np.float64)[:, None] * sw.astype(np.float64)))
    got = host(c)
    assert np.array_equal(got[:, :n], P.r32(y + bias.astype(np.float64)).astype(np.float32)) and np.all(got[:, n:] == 7.0)


def test_scales_that_are_not_numbers_of_pairs_of_ctas(cuda):
    rng = np.random.default_rng(5)
    m, n, k = 300, 4900, 100
    a, sa, w, sw = _inputs(rng, m, n, k)
    sa[[1, 200, 299]], sw[[5, 4899]], sw[6] = (np.inf, np.nan, -np.inf), np.nan, 0.0
    a[1] = 0
    with np.errstate(invalid="ignore"):
        want = _expected(a, sa, w, sw, None)
    got = _run(cuda, a, sa, w, sw, None, m, n, k)
    assert np.array_equal(got, want, equal_nan=True) and np.isfinite(np.delete(got, (1, 200, 299), 0)[:, 7:4899]).all()
