"""The paged 4-bit cache where calls are large enough to take the forms for many rows: appends whose warps take four blocks
of heads, and evictions whose CTAs read slices too long to keep. Bytes and positions are equal."""
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


def _ints(torch, x):
    return dev(torch, np.asarray(x).astype(np.int32))


# kv heads above two blocks of a warp's heads, and 64 heads of rows for each SM: every width of a head, with the last of its
# lanes without a group, head counts that four blocks do not divide, and every form of the rotation
HEADS = [(17, 32), (19, 20), (40, 4), (9, 64), (23, 48), (5, 128), (7, 96), (16, 128), (3, 256), (5, 160), (4, 132), (10, 224)]
FORMS = [(None, False, 0), ("all", False, 0), ("half", False, 0), ("all", True, 0), ("half", True, 0), ("all", True, 1),
         ("half", False, 3), (None, False, 1)]  # dims that turn, halves, floats that K lies off 16 bytes


@pytest.mark.parametrize("kv,hd", HEADS)
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_large_appends(cuda, kv, hd, form):
    torch = cuda
    part, halves, off = FORMS[form]
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    rng = np.random.default_rng(100 * form + kv + hd)
    rows = 64 * sms // kv + 1 + form
    page, seqs, mass = (16, 7, 64)[form % 3], 3, form % 2 == 0
    width = rows // seqs // page + 2
    table = rng.permutation(seqs * width).reshape(seqs, width)
    pool = P4.Pool(torch, seqs * width, page, kv, hd, table, form % 4 == 1, form % 3, fill=77, mass=mass)
    seq = np.arange(rows) % seqs
    pos = np.arange(rows) // seqs
    pad = rng.random(rows) < 0.1
    pos[pad] = -1
    ld = 2 * kv * hd + 4 * (form % 3)
    x = rng.normal(size=rows * ld + off).astype(np.float32)
    r = x[off:].reshape(rows, ld)
    flat = r[:, : 2 * kv * hd]
    odd = rng.random(flat.shape) < 1e-3
    flat[odd] = rng.choice(np.float32([np.nan, np.inf, -np.inf, 3e38, 0.0, 1e-7]), int(odd.sum()))
    flat[rng.random(rows) < 0.02] = 0.0
    flat[rng.random(rows) < 0.02] *= np.float32(1e-5)
    flat[rng.random(rows) < 0.02, kv * hd:] = 40000.0
    cos = sin = rp = None
    live = pos >= 0
    body = x[off:].reshape(rows, ld).astype(np.float64)
    K = body[:, : kv * hd].reshape(rows, kv, hd).copy()
    V = body[:, kv * hd: 2 * kv * hd].reshape(rows, kv, hd)
    if part:
        rot = hd if part == "all" else hd // 2 // 2 * 2
        cos, sin = P.tables(width * page, rot)
        c, s = dev(torch, cos), dev(torch, sin)
        rp = P4.rope(c, s, halves)
        # a product with an infinity or with what passes fp32 has no 64-bit restatement here: only finite K turns
        K[~np.isfinite(K) | (np.abs(K) > 1e30)] = 1.5
        x[off:].reshape(rows, ld)[:, : kv * hd] = K.reshape(rows, -1)
        K[live] = P4.turn(K[live], pos[live], cos, sin, halves)
    xd, seqd, posd = dev(torch, x), _ints(torch, seq), _ints(torch, pos)
    base = xd.data_ptr() + 4 * off
    arrays = [pool.k, pool.v, pool.kp, pool.vp] + ([pool.mass] if mass else [])
    want = [host(t).copy() for t in arrays]
    _capi.check(P4.append(torch, pool, base, base + 4 * kv * hd, ld, rows, seqd, posd, rp))
    (kq, kst, klo), (vq, vst, vlo) = P4.quantise(K), P4.quantise(V)
    G = pool.G
    at, slot = table[seq[live], pos[live] // page], pos[live] % page
    for w, new, n in ((want[0], P4.pack(kq), 16 * G), (want[1], P4.pack(vq), 16 * G), (want[2], P4.params(kst, klo), G),
                      (want[3], P4.params(vst, vlo), G)):
        if pool.heads_first:
            w[at, :, slot, :n] = new[live]
        else:
            w[at, slot, :, :n] = new[live]
    if mass:
        if pool.heads_first:
            want[4][at, :, slot] = 0.0
        else:
            want[4][at, slot] = 0.0
    for t, w in zip(arrays, want):
        assert np.array_equal(host(t), w)
    back = torch.full((rows, ld), -7.0, device="cuda")
    _capi.check(P4.read(torch, pool, back.data_ptr(), back.data_ptr() + 4 * kv * hd, ld, rows, seqd, posd))
    wb = np.full((rows, ld), -7.0, np.float32)
    wb[live, : kv * hd] = P4.values(kq, kst, klo)[live].reshape(-1, kv * hd).astype(np.float32)
    wb[live, kv * hd: 2 * kv * hd] = P4.values(vq, vst, vlo)[live].reshape(-1, kv * hd).astype(np.float32)
    assert np.array_equal(host(back), wb)


def _masses(rng, shape, kind):
    m = np.exp(2 * rng.normal(size=shape)).astype(np.float32)
    if kind == "ties":
        m = np.float32(rng.integers(0, 4, shape))
    elif kind == "odd":
        pick = rng.random(shape)
        m[pick < 0.3] = np.nan
        m[(pick > 0.3) & (pick < 0.5)] = 0.0
        m[(pick > 0.5) & (pick < 0.6)] = np.inf
        m[(pick > 0.6) & (pick < 0.7)] = -1.0
    return m


# one CTA a head, and eight for one head, with slices above the 24576 positions whose keys a CTA keeps
LONG = [(8, 64, [30000, 24700, 29999, 25000, 30000, 27000, 26001, 30000, 29000, 30000], 24650, 64),
        (8, 16, [30000, 200, 0, 30000, 30000, 30000, 30000, 30000, 30000, 30000], 300, 0),
        (1, 64, [210000], 20000, 128), (1, 257, [230001], 200500, 1)]


@pytest.mark.parametrize("kv,page,lens,budget,recent", LONG)
@pytest.mark.parametrize("kind", ["plain", "ties", "odd"])
def test_evictions_of_long_slices(cuda, kv, page, lens, budget, recent, kind):
    torch = cuda
    lib = _capi.load()
    rng = np.random.default_rng(budget + len(kind))
    hd, seqs, width, new_width = 4, len(lens), -(-max(lens) // page), -(-budget // page)
    pages = seqs * (width + new_width)
    both = rng.permutation(pages).reshape(seqs, width + new_width)
    table, new = both[:, :width].copy(), both[:, width:]
    gone = None
    if kind == "odd":  # a page that is not there: its rows weigh as little as a NaN
        gone = width // 3
        table[0, gone] = pages + 5
    pool = P4.Pool(torch, pages, page, kv, hd, table)
    pool.k.copy_(torch.from_numpy(rng.integers(0, 256, tuple(pool.k.shape)).astype(np.uint8)))
    pool.mass.copy_(torch.from_numpy(_masses(rng, tuple(pool.mass.shape), kind)))
    k0, m0 = host(pool.k).copy(), host(pool.mass).copy()
    new_lens = torch.full((seqs,), 99, dtype=torch.int32, device="cuda")
    kept = torch.full((seqs, kv, budget), 99, dtype=torch.int32, device="cuda")
    _capi.check(P4.evict(torch, pool, _ints(torch, lens), budget, recent, _ints(torch, new), new_lens, kept))
    assert lib.jyc_paged_error(1) == (2 if gone is not None else 0)
    assert np.array_equal(host(new_lens), np.minimum(lens, budget))
    got, k1, m1 = host(kept), host(pool.k), host(pool.mass)
    for b, n in enumerate(lens):
        at = np.arange(n)
        page_of = table[b, at // page]
        there = page_of < pages
        m = np.full((n, kv), np.nan, np.float32)
        m[there] = m0[page_of[there], at[there] % page]
        for h in range(kv):
            rows = P4.kept_rows(m[:, h], n, budget, recent)
            assert np.array_equal(got[b, h, : len(rows)], rows) and np.all(got[b, h, len(rows):] == -1)
            to = np.arange(len(rows))
            ok = there[rows]
            dp, ds = new[b, to[ok] // page], to[ok] % page
            sp, ss = page_of[rows[ok]], rows[ok] % page
            assert np.array_equal(k1[dp, ds, h], k0[sp, ss, h])
            assert np.array_equal(m1[dp, ds, h], m0[sp, ss, h], equal_nan=True)


def test_a_captured_fork_and_join_replays(cuda):
    """One graph whose calls run on two streams that part and meet, behind copies and clears: each call's first kernel may
    start while the last one of its stream ends, and waits for all that it follows."""
    torch = cuda
    lib = _capi.load()
    rng = np.random.default_rng(51)
    seqs, hidden, H, kv, hd, page, width, budget = 3, 640, 8, 2, 64, 16, 40, 100
    wide = (H + 2 * kv) * hd
    pages = seqs * (width + 7)
    both = rng.permutation(pages).reshape(seqs, width + 7)
    w = dev(torch, rng.integers(-127, 128, (wide, hidden)).astype(np.int8))
    ws = dev(torch, rng.uniform(1e-3, 2e-3, wide).astype(np.float32))
    cos, sin = P.tables(1000, hd)
    c, s = dev(torch, cos), dev(torch, sin)
    rp = P4.rope(c, s, True)
    newd = _ints(torch, both[:, width:])
    x, lens, turn = torch.zeros(seqs, hidden, device="cuda"), _ints(torch, [1] * seqs), _ints(torch, [0] * seqs)

    class Side:
        def __init__(self):
            self.pool = P4.Pool(torch, pages, page, kv, hd, both[:, :width])
            self.pool.put_random(np.random.default_rng(1), None)
            self.other = P4.Pool(torch, pages, page, kv, hd, both[:, :width])
            self.other.put_random(np.random.default_rng(2), None)
            self.mass = torch.rand(tuple(self.pool.mass.shape), generator=torch.Generator("cuda").manual_seed(3), device="cuda")
            self.xq, self.xs = torch.zeros(seqs, hidden, dtype=torch.int8, device="cuda"), torch.zeros(seqs, device="cuda")
            self.x, self.qkv = torch.zeros(seqs, hidden, device="cuda"), torch.zeros(seqs, wide, device="cuda")
            self.out, self.far = (torch.zeros(seqs, H * hd, device="cuda") for _ in range(2))
            self.nl, self.pos = (torch.zeros(seqs, dtype=torch.int32, device="cuda") for _ in range(2))
            self.kept = torch.zeros(seqs, kv, budget, dtype=torch.int32, device="cuda")
            self.work = P4.workspace(torch, seqs, H, kv, hd, width * page)
            self.aside = torch.cuda.Stream()

        def step(self):
            main, aside = torch.cuda.current_stream(), self.aside
            self.x.copy_(x)  # a copy, then a call
            _capi.check(lib.jyc_quantize_rows_i8(self.x.data_ptr(), hidden, seqs, hidden, self.xq.data_ptr(), hidden,
                                                 self.xs.data_ptr(), main.cuda_stream))
            _capi.check(lib.jyc_matmul_i8(self.xq.data_ptr(), hidden, self.xs.data_ptr(), w.data_ptr(), hidden, ws.data_ptr(), None,
                                          self.qkv.data_ptr(), wide, seqs, wide, hidden, main.cuda_stream))
            aside.wait_stream(main)  # both streams read the products from here on
            with torch.cuda.stream(aside):
                self.other.mass.copy_(self.mass)
                _capi.check(P4.attend(torch, self.other, self.qkv, self.far, H, lens, rp, turn))
                _capi.check(P4.evict(torch, self.other, lens, budget, 8, newd, self.nl, self.kept))
            self.pos.copy_(lens)
            self.pos.sub_(1)
            k = self.qkv.data_ptr() + 4 * H * hd
            _capi.check(P4.append(torch, self.pool, k, k + 4 * kv * hd, wide, seqs, None, self.pos, rp, turn))
            self.pool.mass.zero_()
            _capi.check(P4.attend(torch, self.pool, self.qkv, self.out, H, lens, rp, turn, self.work))
            main.wait_stream(aside)
            # both sides' results are read and written again: the first kernel follows two streams
            _capi.check(lib.jyc_rope_rows(self.far.data_ptr(), H * hd, self.out.data_ptr(), H * hd, 1, H, hd, turn.data_ptr(),
                                          P4.ref(rp), main.cuda_stream))

        def state(self):
            return [host(t).copy() for t in (self.qkv, self.out, self.far, self.nl, self.kept, self.pool.k, self.pool.vp,
                                             self.pool.mass, self.other.k, self.other.kp, self.other.mass)]

    once, again = Side(), Side()
    for side in (once, again):
        side.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again.step()
    for n in ([600, 1, 99], [100, 101, 640], [333, 640, 7]):
        x.normal_()
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        turn.copy_(lens + 300)
        torch.cuda.synchronize()
        once.step()
        torch.cuda.synchronize()
        graph.replay()
        for got, want in zip(again.state(), once.state()):
            assert np.array_equal(got, want, equal_nan=got.dtype.kind == "f")
