"""Attention over the 4-bit pages where keys' V differ by many orders of magnitude: every key counts by its weight, so
the result is bounded by what the weights leave of the values, sum p (|low| + 15 step), group by group and head by head,
and not by the largest value among the keys."""
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


def _weights(qi, qs, k, H, kv, hd):
    w = np.zeros((H, len(k)))
    for h in range(H):
        s = (k[:, h // (H // kv)] @ qi[h]) * qs[h] / np.sqrt(hd)
        w[h] = np.exp(s - s.max())
        w[h] /= w[h].sum()
    return w


def _check(torch, pool, q, out, H, lens):
    """The bound of _paged4.out_tolerance with each head's and group's own weighted sum in the place of the largest value.
    A unit of up to 64 keys goes into the tensor cores only where its largest weight is 2^9 at least and a group's steps and
    lows fit units in which steps are below 2 and lows below 16, steps at 2^-8 at least or lows at 1: the sum is 2^9 * 15 *
    2^-8 > 2^4.9 at least (as 2^5 * 15 * 2^-4 is, the other form: weights from 2^5, steps from 2^-4), and of a key the product of weight and step is off by half of 2^-24 before it is multiplied by up
    to 8, and its weight by as much before it is multiplied by low + 8 step, up to 32: 2^-22 + 2^-20 together, 64 times at
    most 2^-13.6, 2^-18 (64 half steps) of the sum. Steps below 2^-14, next to lows of 1 at least, are off by 2^-25 before
    they are multiplied by up to 8: 4 half steps."""
    hd, kv, G = pool.hd, pool.kv, pool.G
    x = host(q).astype(np.float64).reshape(len(lens), H, hd)
    got = host(out).astype(np.float64).reshape(len(lens), H, hd)
    for b, n in enumerate(lens):
        qi, qs = P.quantise(x[b])
        kq, kst, klo, vq, vst, vlo = pool.rows(b, n)
        v = P4.values(vq, vst, vlo)
        w = _weights(qi, qs, P4.values(kq, kst, klo), H, kv, hd)
        smax = P4.magnitudes(qi, qs, np.abs(kst), klo, hd)
        rel = P4.out_tolerance(n, G, smax, 1.0) + (64 + 4) * P.U24
        for h in range(H):
            g = h // (H // kv)
            size = w[h] @ (np.abs(vlo[:, g]) + 15 * np.abs(vst[:, g]))  # [G]
            tol = size[np.arange(hd) // 32] * rel
            err = np.abs(got[b, h] - w[h] @ v[:, g])
            assert np.all(err <= tol), (b, h, float((err / tol).max()), int((err / tol).argmax()))


# query heads of a unit up to 4, 8 and 16; heads of every size; rows by tensor copies and by others
SHAPES = [(8, 2, 128, 64), (16, 2, 128, 32), (32, 2, 128, 16), (14, 2, 64, 16), (16, 1, 64, 64), (8, 2, 64, 7), (6, 2, 80, 7),
          (24, 1, 256, 16), (12, 3, 192, 32), (10, 2, 100, 5), (4, 4, 32, 16), (40, 2, 128, 64)]


def _pool(torch, rng, kv, hd, page, lens):
    width = -(-max(lens) // page)
    pages = len(lens) * width
    pool = P4.Pool(torch, pages, page, kv, hd, rng.permutation(pages).reshape(len(lens), width), mass=False)
    pool.put_random(rng, None)
    pool.kp.mul_(0.05)
    return pool


def _lower(pool, b, j, bits, hd):
    """Key j of sequence b scores about `bits` (base 2) below the others: queries are positive, half a normal number each."""
    at = pool.where(b, j)
    pool.kp[at][..., 1] -= bits * np.log(2.0) / (0.8 * np.sqrt(hd))


def _run(torch, pool, rng, H, lens):
    q = torch.randn(len(lens), H * pool.hd, device="cuda").abs()
    out = torch.zeros(len(lens), H * pool.hd, device="cuda")
    _capi.check(P4.attend(torch, pool, q, out, H, dev(torch, np.asarray(lens, np.int32))))
    _check(torch, pool, q, out, H, lens)


@pytest.mark.parametrize("H,kv,hd,page", SHAPES)
@pytest.mark.parametrize("bits", [5, 15, 25, 35, 60])
def test_large_values_of_little_weight(cuda, H, kv, hd, page, bits):
    """Three keys at the largest step that append stores, all but unseen by the queries, among keys whose steps are 1e-4 to
    0.1; a fourth is large in one group only."""
    torch = cuda
    rng = np.random.default_rng(1000 * bits + hd + H)
    lens = [70, 400, 1300]
    pool = _pool(torch, rng, kv, hd, page, lens)
    step = 10.0 ** rng.uniform(-4, -1, tuple(pool.vp.shape[:-1]))
    pool.vp.copy_(torch.from_numpy(P4.params(step, -step * rng.uniform(5, 9, step.shape))))
    for b, n in enumerate(lens):
        for j in (0, n // 3, n - 2):
            pool.vp[pool.where(b, j)] = torch.tensor([8736.0, -65504.0], device="cuda").half()
            _lower(pool, b, j, bits, hd)
        at = pool.where(b, n // 2)
        pool.vp[at][..., pool.G - 1, :] = torch.tensor([8736.0, -65504.0], device="cuda").half()
        _lower(pool, b, n // 2, bits, hd)
    _run(torch, pool, rng, H, lens)


@pytest.mark.parametrize("H,kv,hd,page", SHAPES)
@pytest.mark.parametrize("bits", [8, 20, 30, 50])
@pytest.mark.parametrize("first", [False, True])
def test_runs_of_large_values_of_little_weight(cuda, H, kv, hd, page, bits, first):
    """Whole units of keys that are alike and large, hardly seen, before or behind ones that are small."""
    torch = cuda
    rng = np.random.default_rng(2000 * bits + hd + H + first)
    lens = [200, 700]
    pool = _pool(torch, rng, kv, hd, page, lens)
    step = 1e-3 * rng.uniform(1, 4, tuple(pool.vp.shape[:-1]))
    pool.vp.copy_(torch.from_numpy(P4.params(step, -step * rng.uniform(5, 9, step.shape))))
    for b, n in enumerate(lens):
        for j in range(n):
            if (j < n // 2) == first:
                pool.vp[pool.where(b, j)].mul_(2.0 ** 20)
                _lower(pool, b, j, bits, hd)
    _run(torch, pool, rng, H, lens)


@pytest.mark.parametrize("H,kv,hd,page", SHAPES)
def test_values_of_every_kind(cuda, H, kv, hd, page):
    """Steps below fp16's normal numbers, groups of equal values (step 0), of zeros, with offsets far above their steps, and
    of either sign, side by side."""
    torch = cuda
    rng = np.random.default_rng(hd + H)
    lens = [33, 129, 900]
    pool = _pool(torch, rng, kv, hd, page, lens)
    shape = tuple(pool.vp.shape[:-1])
    step = 2.0 ** rng.uniform(-24, 13, shape)
    low = -step * rng.uniform(5, 9, shape)
    kind = rng.integers(0, 8, shape)
    step[kind == 0] = 0.0
    step[kind == 1] = low[kind == 1] = 0.0
    low[kind == 2] = np.minimum(step[kind == 2] * 2000, 60000)
    step[kind == 3] *= -1
    step[kind == 4] = 2.0 ** -24
    low = np.clip(low, -65504, 65504)
    pool.vp.copy_(torch.from_numpy(P4.params(step, low)))
    _run(torch, pool, rng, H, lens)


@pytest.mark.parametrize("H,kv,hd,page", SHAPES)
def test_first_key_takes_the_weight_and_holds_nothing(cuda, H, kv, hd, page):
    """The first key scores far above the others and its V is zero or next to it: the result is what the others leave."""
    torch = cuda
    rng = np.random.default_rng(7 * hd + H)
    lens = [90, 1000]
    pool = _pool(torch, rng, kv, hd, page, lens)
    for b in range(2):
        at = pool.where(b, 0)
        pool.vp[at] = 0.0 if b else 1e-5
        _lower(pool, b, 0, -20, hd)
    _run(torch, pool, rng, H, lens)
