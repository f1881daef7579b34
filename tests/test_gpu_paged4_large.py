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
