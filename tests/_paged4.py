"""Paged 4-bit cache: plain 64-bit forms and device buffers for the tests."""
from __future__ import annotations

import ctypes as C

import numpy as np

from _paged import U24, ptr, r32
from jieyu_b200 import _capi


def groups(hd: int) -> int:
    return -(-hd // 32)


def r16(x):
    """A 64-bit value (of an fp32 number within fp16's range) rounded to fp16, as a 64-bit number."""
    return x.astype(np.float32).astype(np.float16).astype(np.float64)


def turn(x, pos, cos, sin, halves):
    """x [rows][heads][hd] by its row's position, each pair in its place: one product rounded to fp32, then a
    fused sum rounded to fp32."""
    out = np.array(x, np.float64)
    half = cos.shape[1]
    for j in range(half):
        i0, i1 = (j, j + half) if halves else (2 * j, 2 * j + 1)
        c, s = cos[pos, j].astype(np.float64)[:, None], sin[pos, j].astype(np.float64)[:, None]
        a, b = np.array(x[:, :, i0], np.float64), np.array(x[:, :, i1], np.float64)
        out[:, :, i0] = r32(a * c - r32(b * s))
        out[:, :, i1] = r32(a * s + r32(b * c))
    return out


def quantise(x):
    """x [..][hd] (64-bit values of fp32 numbers) as q [..][hd] with step and low [..][G]."""
    hd = x.shape[-1]
    q, steps, lows = np.zeros(x.shape), [], []
    with np.errstate(invalid="ignore", over="ignore"):
        for d in range(0, hd, 32):
            g = x[..., d: d + 32]
            none = np.isnan(g).all(-1)
            lo = np.clip(np.where(none, 0.0, np.where(np.isnan(g), np.inf, g).min(-1)), -65504.0, 65504.0)
            hi = np.clip(np.where(none, 0.0, np.where(np.isnan(g), -np.inf, g).max(-1)), -65504.0, 65504.0)
            low, step = r16(lo), r16(r32(r32(hi - lo) / 15.0))
            inv = np.where(step > 0, r32(1.0 / np.where(step > 0, step, 1.0)), 0.0)
            v = r32(r32(g - low[..., None]) * inv[..., None])
            q[..., d: d + 32] = np.rint(np.clip(np.where(np.isnan(v), 0.0, v), 0, 15))
            steps.append(step)
            lows.append(low)
    return q, np.stack(steps, -1), np.stack(lows, -1)


def values(q, step, low):
    """What stored numbers stand for, unrounded."""
    at = np.arange(q.shape[-1]) // 32
    return low[..., at] + step[..., at] * q


def pack(q):
    """Bytes [..][16 G] of whole numbers q [..][hd]."""
    hd = q.shape[-1]
    full = np.zeros(q.shape[:-1] + (32 * groups(hd),), np.uint8)
    full[..., :hd] = q.astype(np.uint8)
    full = full.reshape(q.shape[:-1] + (groups(hd), 2, 16))
    return (full[..., 0, :] | full[..., 1, :] << 4).reshape(q.shape[:-1] + (16 * groups(hd),))


def params(step, low):
    """fp16 pairs [..][G][2]."""
    return np.stack((step, low), -1).astype(np.float16)


def unpack(b, hd):
    g = b.reshape(b.shape[:-1] + (-1, 1, 16))
    return np.concatenate((g & 15, g >> 4), -2).reshape(b.shape[:-1] + (-1,))[..., :hd].astype(np.float64)


def attention(q, qs, k, v):
    """One sequence: q [H][hd] whole numbers with scales [H], k and v [n][KV][hd] values; out [H][hd] and the keys'
    weights summed over each kv head's query heads [n][KV]."""
    H, hd = q.shape
    KV = k.shape[1]
    out, mass = np.zeros((H, hd)), np.zeros((k.shape[0], KV))
    for h in range(H):
        g = h // (H // KV)
        s = (k[:, g] @ q[h]) * qs[h] / np.sqrt(hd)
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h] = p @ v[:, g]
        mass[:, g] += p
    return out, mass


def rounding(n, G, smax, group=1):
    """Relative rounding of a softmax weight in fp32, in half steps of 1: a score sums 2 G products that were rounded
    as they were added, each bounded by smax (the scores' sum of magnitudes), then takes at most 6 more roundings; all
    of it enters the weight and the sum of weights. exp is off by at most 4 half steps, twice, and the sum of weights
    by one for each of a warp's units of 32 keys and 64 in one of them, a few for joining the parts and dividing; a
    sum over `group` heads adds one each."""
    return U24 * (2 * (2 * G + 6) * smax + 8 + 64 + (n / 32 + 1) + 16 + group)


def out_tolerance(n, G, smax, vmax):
    """A weight's rounding, then weights as two fp16 halves (2^-22: 4 half steps), times a step as two halves (4 more),
    sums inside a unit of at most 64 steps (the tensor cores may truncate), one rounding for each unit and part; vmax
    bounds |low| + 15 step."""
    return vmax * (rounding(n, G, smax) + U24 * (4 + 4 + 64 + (n / 32 + 1) + 16))


def magnitudes(q, qs, step, low, hd):
    """The largest sum of magnitudes that a score is made of: keys' params [n][KV][G], q [H][hd]."""
    G, KV = step.shape[-1], step.shape[1]
    H = q.shape[0]
    worst = 0.0
    for h in range(H):
        g = h // (H // KV)
        pad = np.zeros(32 * G)
        pad[:hd] = np.abs(q[h])
        whole = pad.reshape(G, 32).sum(-1)
        worst = max(worst, ((15 * step[:, g] + np.abs(low[:, g])) @ whole).max() * qs[h] / np.sqrt(hd))
    return worst


class Pool:
    """A 4-bit cache of pages on the device, in either order, with `gap` spare heads' room behind each row."""

    def __init__(self, torch, pages, page, kv, hd, table, heads_first=False, gap=0, fill=0, mass=True):
        self.torch, self.page, self.kv, self.hd, self.heads_first = torch, page, kv, hd, heads_first
        G = self.G = groups(hd)
        a, b = (kv, page) if heads_first else (page, kv)
        self.k = torch.full((pages, a, b, 16 * (G + gap)), fill, dtype=torch.uint8, device="cuda")
        self.v = torch.full_like(self.k, fill)
        self.kp = torch.full((pages, a, b, G + gap, 2), float(fill), dtype=torch.float16, device="cuda")
        self.vp = torch.full_like(self.kp, float(fill))
        self.mass = torch.full((pages, a, b), float(fill), device="cuda") if mass else None
        self.table_host = np.ascontiguousarray(table, np.int32)
        self.table = torch.from_numpy(self.table_host).cuda()
        i, j = (2, 1) if heads_first else (1, 2)
        m = self.kp.stride() if not mass else self.mass.stride()
        self.desc = _capi.KVPagesQ4(
            self.k.data_ptr(), self.kp.data_ptr(), self.v.data_ptr(), self.vp.data_ptr(), ptr(self.mass), pages, page,
            self.k.stride(0), self.k.stride(i), self.k.stride(j), self.kp.stride(0) // 2, self.kp.stride(i) // 2,
            self.kp.stride(j) // 2, *((m[0], m[i], m[j]) if mass else (0, 0, 0)))

    def where(self, seq, pos, head=slice(None), table=None):
        table = self.table_host if table is None else table
        page, slot = int(table[seq, pos // self.page]), pos % self.page
        return (page, head, slot) if self.heads_first else (page, slot, head)

    def put_random(self, rng, lens, scale=1.0):
        """Random rows everywhere: the whole pool at once."""
        torch, G, hd = self.torch, self.G, self.hd
        for x, p in ((self.k, self.kp), (self.v, self.vp)):
            shape = tuple(x.shape[:-1])
            x[..., : 16 * G] = torch.from_numpy(pack(rng.integers(0, 16, shape + (hd,)))).cuda()
            step = scale * rng.uniform(0.05, 0.3, shape + (G,))
            p[..., :G, :] = torch.from_numpy(params(step, -step * rng.uniform(5, 9, shape + (G,)))).cuda()

    def rows(self, seq, n, table=None):
        """Host values of positions 0..n-1: q, step, low of K, then of V, [n][kv][..]."""
        table = self.table_host if table is None else table
        at = np.arange(n)
        page, slot = self.torch.from_numpy(table[seq, at // self.page].astype(np.int64)).cuda(), self.torch.from_numpy(
            at % self.page).cuda()
        out = []
        for x, p in ((self.k, self.kp), (self.v, self.vp)):
            xs = x[page, :, slot] if self.heads_first else x[page, slot]
            ps = p[page, :, slot] if self.heads_first else p[page, slot]
            ps = ps[..., : self.G, :].cpu().numpy().astype(np.float64)
            out += [unpack(xs[..., : 16 * self.G].cpu().numpy(), self.hd), ps[..., 0], ps[..., 1]]
        return out

    def masses(self, seq, n, table=None):
        table = self.table_host if table is None else table
        at = np.arange(n)
        m = self.mass.cpu().numpy()
        page, slot = table[seq, at // self.page], at % self.page
        return m[page, :, slot] if self.heads_first else m[page, slot]


def rope(cos, sin, halves, length=None):
    return _capi.Rope(cos.data_ptr(), sin.data_ptr(), cos.shape[0] if length is None else length, 2 * cos.shape[1],
                      _capi.JYC_ROPE_HALVES if halves else _capi.JYC_ROPE_PAIRS)


def ref(x):
    return None if x is None else C.byref(x)


def workspace(torch, seqs, H, KV, hd, capacity, fill=255):
    n = _capi.load().jyc_attention_paged_q4_workspace(seqs, H, KV, hd, capacity)
    assert n > 0
    return torch.full((n,), fill, dtype=torch.uint8, device="cuda")


def stream_of(torch):
    return torch.cuda.current_stream().cuda_stream


def append(torch, pool, K, V, ld, rows, seq, pos, rp=None, rope_pos=None, stream=None):
    return _capi.load().jyc_kv_append_paged_q4(
        K, V, ld, rows, pool.kv, pool.hd, ptr(seq), ptr(pos), ptr(pool.table), pool.table.shape[1],
        pool.table.shape[0], ref(rp), ptr(rope_pos), C.byref(pool.desc), stream_of(torch) if stream is None else stream)


def read(torch, pool, K, V, ld, rows, seq, pos, table=None, stream=None):
    t = pool.table if table is None else table
    return _capi.load().jyc_kv_read_paged_q4(K, V, ld, rows, pool.kv, pool.hd, ptr(seq), ptr(pos), ptr(t), t.shape[1],
                                             t.shape[0], C.byref(pool.desc),
                                             stream_of(torch) if stream is None else stream)


def attend(torch, pool, q, out, H, lens, rp=None, rope_pos=None, work=None, seqs=None, stream=None, table=None):
    t = pool.table if table is None else table
    return _capi.load().jyc_attention_paged_q4(
        ptr(q), q.stride(0), ptr(out), out.stride(0), H, pool.kv, pool.hd, ptr(lens), ptr(t), t.shape[1],
        len(lens) if seqs is None else seqs, ref(rp), ptr(rope_pos), C.byref(pool.desc), ptr(work),
        0 if work is None else work.numel(), stream_of(torch) if stream is None else stream)


def evict(torch, pool, lens, budget, recent, new_table, new_lens, kept, stream=None):
    return _capi.load().jyc_kv_evict_paged_q4(
        ptr(lens), budget, recent, pool.kv, pool.hd, ptr(pool.table), pool.table.shape[1], len(lens), ptr(new_table),
        new_table.shape[1], ptr(new_lens), ptr(kept), C.byref(pool.desc), stream_of(torch) if stream is None else stream)


def kept_rows(mass, n, budget, recent):
    """Positions that one kv head of a sequence of n rows keeps: mass [n] fp32."""
    if n <= budget:
        return np.arange(n)
    old = np.arange(n - recent)
    m = np.where(np.isnan(mass[old]), -np.inf, mass[old].astype(np.float64))
    nan = np.isnan(mass[old])
    best = np.lexsort((old, nan, -m))[: budget - recent]
    return np.concatenate((np.sort(old[best]), np.arange(n - recent, n)))
