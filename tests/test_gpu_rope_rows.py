"""jyc_rope_rows on the device: bit for bit against the rounding that the 64-bit form spells out."""
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


def _turn(torch, x, y, ldx, ldy, rows, heads, hd, pos, rp, stream=None):
    return _capi.load().jyc_rope_rows(x, ldx, y, ldy, rows, heads, hd, P.ptr(pos), P4.ref(rp),
                                      P4.stream_of(torch) if stream is None else stream)


SHAPES = [  # heads, hd, rot, extra floats of a row, offset in floats
    (40, 128, 128, 0, 0), (3, 64, 32, 4, 0), (5, 80, 40, 0, 4), (1, 4, 2, 0, 0), (7, 36, 34, 1, 0), (2, 256, 250, 0, 1),
    (3, 33, 20, 0, 0), (9, 96, 96, 8, 0), (2, 128, 64, 0, 2),
]


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("heads,hd,rot,extra,off", SHAPES)
@pytest.mark.parametrize("rows,in_place", [(1, False), (19, True), (130, False)])
def test_rows(cuda, heads, hd, rot, extra, off, halves, rows, in_place):
    torch = cuda
    rng = np.random.default_rng(rows * 7 + hd)
    n = 97
    cos, sin = P.tables(n, rot)
    ld = heads * hd + extra
    x = rng.normal(size=off + rows * ld).astype(np.float32)
    pos = rng.integers(0, n, rows)
    if rows > 4:
        pos[rng.permutation(rows)[:3]] = (-1, -(1 << 31), -7)
        pos[rng.integers(0, rows)] = n - 1
    xd, yd = dev(torch, x), torch.full((off + rows * ld,), -5.0, device="cuda")
    c, s = dev(torch, cos), dev(torch, sin)
    to = xd if in_place else yd
    _capi.check(_turn(torch, xd.data_ptr() + 4 * off, to.data_ptr() + 4 * off, ld, ld, rows, heads, hd,
                      dev(torch, pos.astype(np.int32)), P4.rope(c, s, halves)))
    want = (x if in_place else np.full_like(x, -5.0)).copy()
    body = x[off:].reshape(rows, ld)[:, : heads * hd].reshape(rows, heads, hd)
    live = pos >= 0
    want[off:].reshape(rows, ld)[live, : heads * hd] = P4.turn(body[live], pos[live], cos, sin, halves).reshape(
        live.sum(), -1)
    assert np.array_equal(host(to), want)
    if not in_place:
        assert np.array_equal(host(xd), x)


def test_positions_behind_the_tables(cuda):
    torch = cuda
    lib = _capi.load()
    cos, sin = P.tables(8, 64)
    c, s = dev(torch, cos), dev(torch, sin)
    x = torch.randn(4, 2 * 64, device="cuda")
    y = torch.zeros_like(x)
    pos = torch.tensor([0, 8, 7, 2**31 - 1], dtype=torch.int32, device="cuda")
    _capi.check(_turn(torch, x.data_ptr(), y.data_ptr(), 128, 128, 4, 2, 64, pos, P4.rope(c, s, True)))
    assert lib.jyc_paged_error(1) == 4
    got = host(y)
    assert np.all(got[[1, 3]] == 0.0) and np.all(np.abs(got[[0, 2]]).sum(-1) > 0)


def test_halves_equal_pairs_of_reordered_dims(cuda):
    """Both layouts turn the same pairs: a head whose dims are reordered gives the reordered result."""
    torch = cuda
    rng = np.random.default_rng(2)
    rows, heads, hd = 11, 3, 64
    cos, sin = P.tables(50, hd)
    c, s = dev(torch, cos), dev(torch, sin)
    x = rng.normal(size=(rows, heads, hd)).astype(np.float32)
    order = np.stack((np.arange(hd // 2), np.arange(hd // 2) + hd // 2), -1).reshape(-1)
    pos = dev(torch, rng.integers(0, 50, rows).astype(np.int32))
    got = []
    for v, halves in ((x, True), (x[..., order], False)):
        xd = dev(torch, v)
        y = torch.empty_like(xd)
        _capi.check(_turn(torch, xd.data_ptr(), y.data_ptr(), heads * hd, heads * hd, rows, heads, hd, pos,
                          P4.rope(c, s, halves)))
        got.append(host(y))
    assert np.array_equal(got[0][..., order], got[1])


def test_graph_and_stream(cuda):
    torch = cuda
    rows, heads, hd = 33, 4, 128
    cos, sin = P.tables(64, hd)
    c, s = dev(torch, cos), dev(torch, sin)
    rp = P4.rope(c, s, False)
    x, y = torch.randn(rows, heads * hd, device="cuda"), torch.zeros(rows, heads * hd, device="cuda")
    pos = torch.zeros(rows, dtype=torch.int32, device="cuda")
    _capi.check(_turn(torch, x.data_ptr(), y.data_ptr(), heads * hd, heads * hd, rows, heads, hd, pos, rp))
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        _capi.check(_turn(torch, x.data_ptr(), y.data_ptr(), heads * hd, heads * hd, rows, heads, hd, pos, rp,
                          torch.cuda.current_stream().cuda_stream))
    for shift in (3, 40):
        pos.fill_(shift)
        x.normal_()
        graph.replay()
        want = P4.turn(host(x).reshape(rows, heads, hd), np.full(rows, shift), cos, sin, False)
        assert np.array_equal(host(y).reshape(rows, heads, hd), want.astype(np.float32))
