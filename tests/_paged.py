"""Paged int8 cache and batch sampling: plain 64-bit forms and device buffers for the tests."""
from __future__ import annotations

import ctypes as C

import numpy as np

from jieyu_b200 import _capi

U24 = 2.0 ** -24  # half a step of fp32, relative


def r32(x):
    """A 64-bit result rounded to fp32, as a 64-bit number."""
    with np.errstate(over="ignore"):
        return np.asarray(x, np.float64).astype(np.float32).astype(np.float64)


def slot_of(p: int, half: int) -> int:
    """Where rotated pair p is stored (rope_pos's order): 2,3 <-> 4,5 in every full group of 8."""
    return p - p % 8 + (0, 1, 4, 5, 2, 3, 6, 7)[p % 8] if p - p % 8 + 8 <= half else p


def rotate(x, pos, cos, sin):
    """x [rows][heads][hd] (64-bit values of fp32 inputs) by its row's position: one product
    rounded to fp32, then a fused sum rounded to fp32."""
    out = np.empty_like(x)
    half = x.shape[-1] // 2
    for p in range(half):
        o = slot_of(p, half)
        c, s = cos[pos, p].astype(np.float64)[:, None], sin[pos, p].astype(np.float64)[:, None]
        a, b = x[:, :, 2 * p], x[:, :, 2 * p + 1]
        out[:, :, 2 * o] = r32(a * c - r32(b * s))
        out[:, :, 2 * o + 1] = r32(a * s + r32(b * c))
    return out


def quantise(x):
    """kv_pack_q8's rule over the last axis: whole numbers and the fp32 scale, as 64-bit values."""
    with np.errstate(invalid="ignore", divide="ignore"):
        amax = np.max(np.where(np.isnan(x), 0.0, np.abs(x)), axis=-1, keepdims=True)
        big = amax > np.float64(np.float32(1e-8))
        inv = np.where(big, r32(127.0 / np.where(big, amax, 1.0)), 0.0)
        scale = np.where(big, r32(amax / 127.0), 0.0)
        v = r32(x * inv)
        return np.rint(np.where(np.isnan(v), 0.0, np.clip(v, -127, 127))), scale[..., 0]


def attention(q, qs, k, ks, v, vs, scale=None):
    """One sequence: q [H][hd] whole numbers with scales [H], k and v [n][KV][hd] with scales [n][KV]."""
    H, hd = q.shape
    KV = k.shape[1]
    out = np.zeros((H, hd))
    for h in range(H):
        g = h // (H // KV)
        s = (k[:, g] @ q[h]) * ks[:, g] * qs[h] / np.sqrt(hd)
        p = np.exp(s - s.max())
        out[h] = ((p / p.sum()) * vs[:, g]) @ v[:, g]
    return out


def attention_tolerance(n, smax, vmax):
    """Worst-case rounding of an fp32 kernel that sums blocks of 32 keys: scores carry at most 8
    roundings (relative, so 8 smax half steps absolute, entering p and the sum: twice), exp 4 half
    steps twice, a weight as two fp16 halves 2^-22, sums inside a block of 32 keys at most 64 steps
    (the tensor cores may truncate) and one rounding per block in numerator and denominator, a few
    more for joining the parts and the division."""
    return vmax * U24 * (2 * 8 * smax + 2 * 4 + 4 + 2 * 64 + 2 * (n / 32 + 1) + 16)


class Pool:
    """A cache of pages on the device, in either order, and its page table."""

    def __init__(self, torch, pages, page, kv, hd, table, heads_first=False, gap=0, fill=None):
        self.torch, self.page, self.kv, self.hd, self.heads_first = torch, page, kv, hd, heads_first
        a, b = (kv, page) if heads_first else (page, kv)
        self.k8 = torch.zeros(pages, a, b, hd + gap, dtype=torch.int8, device="cuda")
        self.v8 = torch.zeros_like(self.k8)
        self.ks = torch.zeros(pages, a, b, device="cuda")
        self.vs = torch.zeros_like(self.ks)
        if fill is not None:
            self.k8.fill_(fill)
            self.v8.fill_(fill)
            self.ks.fill_(float("nan"))
            self.vs.fill_(float("nan"))
        self.table_host = np.ascontiguousarray(table, np.int32)
        self.table = torch.from_numpy(self.table_host).cuda()
        i, j = (2, 1) if heads_first else (1, 2)
        self.desc = _capi.KVPages(self.k8.data_ptr(), self.ks.data_ptr(), self.v8.data_ptr(), self.vs.data_ptr(),
                                  pages, page, self.k8.stride(0), self.k8.stride(i), self.k8.stride(j),
                                  self.ks.stride(0), self.ks.stride(i), self.ks.stride(j))

    def at(self, seq, pos):
        """(K bytes, K scale, V bytes, V scale) [kv][..] of one position, from a host copy."""
        page, slot = int(self.table_host[seq, pos // self.page]), pos % self.page
        idx = (page, slice(None), slot) if self.heads_first else (page, slot)
        return tuple(t[idx].cpu().numpy() for t in (self.k8[..., : self.hd], self.ks, self.v8[..., : self.hd], self.vs))

    def rows(self, seq, n):
        """Host copies of positions 0..n-1: k [n][kv][hd], ks [n][kv], v, vs as 64-bit values."""
        pages = self.table_host[seq, : -(-n // self.page)].astype(np.int64)
        out = []
        for t in (self.k8[..., : self.hd], self.ks, self.v8[..., : self.hd], self.vs):
            x = t[self.torch.from_numpy(pages).cuda()].cpu().numpy().astype(np.float64)
            if self.heads_first:
                x = np.swapaxes(x, 1, 2)
            out.append(x.reshape((-1,) + x.shape[2:])[:n])
        return out

    def put_random(self, rng, seq, n):
        """Random rows at positions 0..n-1 of a sequence."""
        torch = self.torch
        for j in range(0, n, self.page):
            m = min(self.page, n - j)
            page = int(self.table_host[seq, j // self.page])
            for t8, ts in ((self.k8, self.ks), (self.v8, self.vs)):
                q = np.clip(np.rint(rng.normal(0, 45, (m, self.kv, self.hd))), -127, 127).astype(np.int8)
                s = rng.uniform(0.005, 0.03, (m, self.kv)).astype(np.float32)
                if self.heads_first:
                    t8[page, :, :m, : self.hd] = torch.from_numpy(np.ascontiguousarray(q.swapaxes(0, 1))).cuda()
                    ts[page, :, :m] = torch.from_numpy(np.ascontiguousarray(s.T)).cuda()
                else:
                    t8[page, :m, :, : self.hd] = torch.from_numpy(q).cuda()
                    ts[page, :m] = torch.from_numpy(s).cuda()


def tables(n, hd, theta=1e4):
    j = np.arange(hd // 2)
    ang = np.arange(n)[:, None] * theta ** (-2.0 * j / hd)
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def ptr(t):
    return None if t is None else t.data_ptr()


def workspace(torch, seqs, H, KV, hd, fill=255):
    n = _capi.load().jyc_attention_paged_q8_workspace(seqs, H, KV, hd)
    assert n > 0
    return torch.full((n,), fill, dtype=torch.uint8, device="cuda")


def attend(torch, pool, q, out, H, lens, cos=None, sin=None, work=None, seqs=None, stream=None, rope_len=None):
    seqs = len(lens) if seqs is None else seqs
    stream = torch.cuda.current_stream().cuda_stream if stream is None else stream
    return _capi.load().jyc_attention_paged_q8(
        ptr(q), q.stride(0), ptr(out), out.stride(0), H, pool.kv, pool.hd, ptr(lens), ptr(pool.table),
        pool.table.shape[1], seqs, ptr(cos), ptr(sin), (0 if cos is None else cos.shape[0]) if rope_len is None else
        rope_len, C.byref(pool.desc), ptr(work), 0 if work is None else work.numel(), stream)


# ---- sampling -------------------------------------------------------------

CUT = 2.0 ** -40


def weights(l, T):
    l = np.where(np.isnan(l), -np.inf, l.astype(np.float64)) + 0.0
    top = l.max()
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(l == top, 1.0, np.where(l == -np.inf, 0.0, np.exp((l - top) / T)))
    w[w < CUT] = 0.0
    return l, w


def picks(l, T, k, p, mp, u):
    """(ids that the definition allows for this row, their probabilities): more than one where a sum
    lies within the fixed-point rounding of a border (half a step of 2^-42 per token, and a
    relative 2^-44 of exp)."""
    V = len(l)
    l64 = np.where(np.isnan(l), -np.inf, l.astype(np.float64))
    if l64.max() == -np.inf:
        return {-1: 0.0}
    if not T > 0:
        return {int(np.argmax(l64)): 1.0}
    l64, w = weights(l, np.float64(np.float32(T)))
    order = np.argsort(-l64, kind="stable")
    if k is not None and 0 < k < V:
        order = order[:k]
    slack = V * 2.0 ** -43 + 2.0 ** -44 * w.sum()
    sets = [order]
    if p is not None and p < 1:
        sums = np.cumsum(w[order])
        need = np.float64(np.float32(p)) * sums[-1]
        ns = {1 + int(np.searchsorted(sums, x, side="left")) for x in (need, need - slack, need + slack)}
        sets = [order[: max(1, min(n, len(order)))] for n in ns]
    found = {}
    for chosen in sets:
        keep = w[chosen] > 0
        if mp is not None:
            keep &= w[chosen] >= min(1.0, np.float64(np.float32(mp)))
        idx = np.sort(chosen[keep])
        sums = np.cumsum(w[idx])
        r = np.float64(np.float32(u)) * sums[-1]
        for x in (r, r - slack, r + slack):
            at = min(int(np.searchsorted(sums, x, side="right")), len(idx) - 1)
            found.setdefault(int(idx[at]), w[idx[at]] / sums[-1])
    return found
