// pick.cu — the next token of every row of a batch: temperature, top-k, top-p
// and min-p filters, then one inverse-CDF draw per row from a given random
// number (beside sample.cuh, which restates the reference's one-row sampler).
//
// Every filter keeps a prefix of the order (logit descending, index ascending),
// so with comp = (order key of the logit, ~index) a kept set is {comp >= tau},
// and weights only decide where the prefix ends. Weights 2^((l - max) log2(e) /
// T) are held as 2^42 fixed point in 64 bits (below 2^-40: zero): their sums
// are the same in any order.
//
// A row belongs to a cluster of 1 to 8 CTAs that exchange through distributed
// shared memory, so one launch serves one row or hundreds. Nothing is sorted.
//   1  the maximum (a greedy row ends here); every lane keeps four maxima.
//   2  a bin of (max - l) / T such that the tokens up to it hold the kept set and
//      are as few as can be told: with top-k from the k-th of those maxima (as
//      many logits are as large), with min-p from min_p itself, with top-p from a
//      bound on the mass of all smaller ones. One pass puts those tokens, in index
//      order, into pools (one per warp), sums all weights and adds the pools' to a
//      histogram of the bins (fp32 shares in fixed point: bounds of 4e-5).
//   3  pools of 4096 tokens in all or fewer: one CTA takes them and ends the row,
//      finding each border by bisection over keys.
//      More: the histogram bounds the running count or mass, so the border lies in
//      one or two bins; their tokens go to one CTA (or are split by exact sums while
//      they are more than 512), which finds the last kept one by sums over digits of
//      the keys. The kept weights are summed by warp, in index order; the warp
//      that the draw falls in walks its tokens.
//   Rows without a filter, with k above 2048, and rows whose pools overflow go
//   through 3 over all their logits instead of the pools.
// Floor: one read of the logits; later passes find them in L2. What is left of
// the time is the chain of passes and exchanges of a row (21 us for one row with
// top-k, 49 with top-p alone); with many rows too: warps wait at barriers more than
// for memory (64 rows of top-p: 5.8 stalls an issue against 1.7), and 42 % of the
// issue slots are busy. They execute 203 instructions per 32 logits over all
// passes; the exact weights of one pass are 22 of them, 11 in double precision.
#include <cooperative_groups.h>

#include <algorithm>

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace jyc {

namespace {

typedef unsigned long long u64;

constexpr int kPickThreads = 512, kPickWarps = kPickThreads / 32;
constexpr int kPickList = 4096;      // tokens that one CTA ends a row with
constexpr int kPickTopK = 2048;      // largest k bounded by maxima: as many as a CTA keeps
constexpr int kPickPool = 1920;      // tokens of a warp's pool: two CTAs share an SM's memory
constexpr int kPickPairs = 256;      // tokens whose top-p is decided by comparing all pairs
constexpr int kPickRank = 512;       // tokens among which one CTA looks for a border
constexpr int kPickGather = 128;     // tokens that a warp gathers before it weighs them
constexpr int kPickDigit = 9;        // bits of a key's digit in that search: a bin a thread
constexpr int kPickBins = 2048, kPickPer = kPickBins / kPickThreads;
constexpr int kPickWide = kPickBins / 2;  // bins of 64-bit sums, in the same memory
constexpr int kPickMaxCluster = 8;
constexpr float kPickSpan = 40.0f;   // powers of two that the bins cover
constexpr double kOne = 0x1p42;      // a weight of 1

__device__ __forceinline__ u64 pick_comp(float l, int idx) {
    return (u64)f32_order_key(l + 0.0f) << 32 | (u64)(0xFFFFFFFFu - (uint32_t)idx);  // -0 as +0
}
__device__ __forceinline__ int pick_index(u64 comp) { return (int)(0xFFFFFFFFu - (uint32_t)comp); }
__device__ __forceinline__ float pick_value(u64 comp) {
    const uint32_t k = (uint32_t)(comp >> 32);
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

__device__ __forceinline__ float pick_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct PickShared {
    union {
        u64 list[kPickList];
        struct {
            u64 first[kPickList / 2];  // a border's tokens, while the totals are in use
            union {
                uint32_t tot[kPickBins];
                u64 wide_tot[kPickWide];
            };
        };
    };
    union {
        uint16_t pool[kPickWarps][kPickPool];  // positions in the warp's part (at most 2^16 logits)
        u64 top[kPickTopK];                    // the top-k, when one CTA ends the row
    };
    ulonglong2 pair[kPickRank];        // comp, metric
    union {
        uint32_t hist[kPickBins];
        u64 wide[kPickWide];
    };
    double pow2[64];                   // 2^(j / 64)
    u64 x[2][kPickMaxCluster];         // exchanges between CTAs, two turns
    u64 x4[kPickMaxCluster][4];
    u64 sums[kPickMaxCluster][kPickWarps];
    u64 red[kPickWarps], red2[kPickWarps];
    u64 tau, border;
    uint32_t count, inside[kPickWarps];
    int b1, b2;
};

// One row, as a CTA sees it.
struct PickRow {
    const float* l;
    int V, v0, v1, w0, w1;  // the CTA's part, the warp's part
    bool vec;
    float mx;
    double c;               // log2(e) / T
    bool endless;           // the maximum is infinite
    float lift, mx_lift;    // places are differences of logits times lift, a power of two: fp32 holds them
    float bin_scale;
    int C, rank, turn;
    int pooled;             // tokens in the warp's pool; -1: the passes go over all logits
    PickShared* s;

    // a logit as the passes take it: under an infinite maximum, 0 where it is infinite too, else -inf
    __device__ __forceinline__ float seen(float x) const { return !endless ? x : x == INFINITY ? 0.0f : -INFINITY; }
    __device__ __forceinline__ float at(int i) const { return seen(__ldg(l + i)); }
    // four logits at i, i + 1, ... < w1 (NaN behind the end)
    __device__ __forceinline__ void load(int i, float (&x)[4]) const {
        if (vec && i + 3 < w1) {
            const float4 q = __ldg(reinterpret_cast<const float4*>(l + i));
            x[0] = q.x;
            x[1] = q.y;
            x[2] = q.z;
            x[3] = q.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = i + j < w1 ? __ldg(l + i + j) : __int_as_float(0x7FC00000);
        }
        if (endless)
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = seen(x[j]);
    }
    // The weight of x in units of 2^-42, a whole number. 2^t by 2^(j / 64) and the series of 2^f: |f| <= 1 / 128,
    // remainder (f ln 2)^5 / 120 < 4e-14
    __device__ __forceinline__ double mass(float x) const {
        const double t = ((double)x - (double)mx) * c;
        const double m = __fma_rn(t, 64.0, 0x1.8p52);
        const int n = __double2loint(m);
        const double f = __fma_rn(m - 0x1.8p52, -1.0 / 64.0, t);
        double p = __fma_rn(f, 0.00961812910762847716, 0.0555041086648215800);
        p = __fma_rn(p, f, 0.240226506959100712);
        p = __fma_rn(p, f, 0.693147180559945309);
        p = __fma_rn(p, f, 1.0) * s->pow2[n & 63];
        const double q = __hiloint2double(__double2hiint(p) + ((n & ~63) << 14) + (42 << 20), __double2loint(p));
        return t >= -40.0 ? (q + 0x1p52) - 0x1p52 : 0.0;  // 0 for NaN and -inf too
    }
    __device__ __forceinline__ u64 weight(float x) const { return (u64)mass(x); }
    // Bins of powers of 2^(40 / 2048), the nearest one: larger logits never lie in a later bin. The place of a
    // logit above -inf among them (0 for the maximum), and its bin.
    __device__ __forceinline__ float place(float x) const {
        return fminf(__fmul_rn(__fmaf_rn(-x, lift, mx_lift), bin_scale), (float)(kPickBins - 1));
    }
    static __device__ __forceinline__ int bin_at(float place) {
        return __float_as_int(__fadd_rn(place, 12582912.0f)) - 0x4B400000;  // 1.5 * 2^23: to the nearest
    }
    __device__ __forceinline__ int bin(float x) const { return bin_at(place(x)); }
    // adds the weight's share of 2^-(bin's middle) to the bin, in units of 1 / unit (fp32: off by less than 1e-5 and
    // half a unit)
    __device__ __forceinline__ void share(float place, float unit) const {
        const float near = __fadd_rn(place, 12582912.0f), off = __fsub_rn(__fsub_rn(near, 12582912.0f), place);
        const float n = __fmul_rn(unit, pick_ex2((kPickSpan / kPickBins) * off));
        atomicAdd(&s->hist[__float_as_int(near) - 0x4B400000], __float2uint_rn(n));
    }
    // f(four logits, their indices, whether there are any) for the warp's tokens, by whole warps: four at a time,
    // so that loads and double-precision chains overlap
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        const int lane = threadIdx.x & 31;
        const bool pools = pooled >= 0;
        const uint16_t* p = s->pool[threadIdx.x >> 5];
        const int end = pools ? pooled : w1;
        float x[4], nx[4];
        int idx[4], nidx[4];
        auto fetch = [&](int i) {  // one step ahead of its use
            if (pools) {
#pragma unroll
                for (int j = 0; j < 4; j++) nidx[j] = i + 32 * j + lane < pooled ? w0 + p[i + 32 * j + lane] : -1;
#pragma unroll
                for (int j = 0; j < 4; j++) nx[j] = nidx[j] >= 0 ? at(nidx[j]) : -INFINITY;
            } else {
                load(i + 4 * lane, nx);
#pragma unroll
                for (int j = 0; j < 4; j++) nidx[j] = i + 4 * lane + j;
            }
        };
        int i = pools ? 0 : w0;
        if (i < end) fetch(i);
        for (; i < end; i += 128) {
            bool is[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                x[j] = nx[j];
                idx[j] = nidx[j];
                is[j] = x[j] > -INFINITY;
            }
            if (i + 128 < end) fetch(i + 128);
            f(x, idx, is);
        }
    }
    __device__ void sync() const {
        if (C > 1)
            cg::this_cluster().sync();
        else
            __syncthreads();
    }
    __device__ PickShared* of(int r) const { return C > 1 ? cg::this_cluster().map_shared_rank(s, r) : s; }
    // v of every CTA (the same in its threads), in s->x[turn][rank of it] after the call
    __device__ const u64* exchange(u64 v) {
        turn ^= 1;
        if ((int)threadIdx.x < C) of(threadIdx.x)->x[turn][rank] = v;
        sync();
        return s->x[turn];
    }
};

template <class F>
__device__ __forceinline__ u64 pick_reduce(u64 v, u64* red, F f) {  // result in every thread
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < kPickWarps; w++) v = f(v, red[w]);
    __syncthreads();
    return v;
}
__device__ __forceinline__ u64 pick_add(u64 a, u64 b) { return a + b; }
__device__ __forceinline__ u64 pick_max(u64 a, u64 b) { return a > b ? a : b; }
__device__ __forceinline__ u64 pick_min(u64 a, u64 b) { return a < b ? a : b; }

// sum over the cluster of one value per thread
__device__ u64 pick_sum(PickRow& r, u64 v) {
    v = pick_reduce(v, r.s->red, pick_add);
    const u64* x = r.exchange(v);
    u64 t = 0ull;
    for (int i = 0; i < r.C; i++) t += x[i];
    return t;
}

// inclusive sum over the block of one value per thread
template <class T>
__device__ __forceinline__ T pick_scan(T v, T* red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    if (lane == 31) red[warp] = v;
    __syncthreads();
    T before = T(0);
    for (int w = 0; w < warp; w++) before += red[w];
    __syncthreads();
    return before + v;
}

// Appends comp to the CTA's list where `take` holds (whole warps call it); s->count counts on past the end.
__device__ __forceinline__ void pick_append(PickShared* s, bool take, u64 comp) {
    const unsigned m = __ballot_sync(0xffffffffu, take);
    if (m == 0u) return;
    const int lane = threadIdx.x & 31;
    uint32_t at = 0u;
    if (lane == 0) at = atomicAdd(&s->count, (uint32_t)__popc(m));
    at = __shfl_sync(0xffffffffu, at, 0) + __popc(m & ((1u << lane) - 1u));
    if (take && at < kPickRank) s->list[at] = comp;
}

// The CTAs' lists (CTA i's of x[step * i] tokens) joined in the first one's, in the CTAs' order, when they are at
// most `most`. Returns their total (-1: too many), the same in every CTA; the list is complete after the call.
__device__ int pick_collect(PickRow& r, const u64* x, int step, int most) {
    u64 total = 0ull, before = 0ull;
    for (int i = 0; i < r.C; i++) {
        if (i < r.rank) before += x[step * i];
        total += x[step * i];
    }
    const uint32_t mine = (uint32_t)x[step * r.rank];
    if (total <= (u64)most && r.rank > 0) {
        u64* to = cg::this_cluster().map_shared_rank(r.s, 0)->list;
        for (uint32_t i = threadIdx.x; i < mine; i += kPickThreads) to[before + i] = r.s->list[i];
    }
    r.sync();
    return total <= (u64)most ? (int)total : -1;
}

// Sums of the CTA's histograms (s->hist, s->wide) in s->tot (s->wide_tot) of every CTA.
template <class T>
__device__ void pick_total(PickRow& r, T* hist, T* tot) {
    constexpr int bins = sizeof(T) == 4 ? kPickBins : kPickWide;
    r.sync();
    if (r.C == 1) {
        for (int b = threadIdx.x; b < bins; b += kPickThreads) tot[b] = hist[b];
        __syncthreads();
        return;
    }
    const int per = bins / r.C;
    for (int i = threadIdx.x; i < per; i += kPickThreads) {
        const int b = r.rank * per + i;
        T n = 0;
        for (int c = 0; c < r.C; c++) n += cg::this_cluster().map_shared_rank(hist, c)[b];
        for (int c = 0; c < r.C; c++) cg::this_cluster().map_shared_rank(tot, c)[b] = n;
    }
    r.sync();
}

// One step of the search below: the members (comps of [*clo, *chi] from tau0 on, of the bins lo_bin .. hi_bin) are split
// into bins of exact sums, and the range shrinks to the bin in which the metric reaches `target` (the last one if none
// does); `up`: the metric above the range. Few rows need it: a call, so that it takes no registers from the others (64 rows
// of top-p 132 us, 139 with the step in line; 256 mixed rows 250 and 261).
__device__ __noinline__ void pick_split(PickRow r, bool by_mass, double target, u64 tau0, int lo_bin, int hi_bin, u64 up,
                                        u64* clo_p, u64* chi_p) {
    constexpr int PER = kPickWide / kPickThreads;
    PickShared* s = r.s;
    const int tid = threadIdx.x;
    const u64 clo = *clo_p, chi = *chi_p;
    int shift = 0;
    while (((chi - clo) >> shift) >= (u64)kPickWide) shift++;
    for (int b = tid; b < kPickWide; b += kPickThreads) s->wide[b] = 0ull;
    if (tid == 0) s->b1 = (double)up >= target ? 0 : kPickWide;
    __syncthreads();
    r.each([&](const float (&x)[4], const int (&idx)[4], const bool (&is)[4]) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const u64 comp = pick_comp(x[j], idx[j]);
            if (!is[j] || comp < tau0 || comp < clo || comp > chi) continue;
            const int b = r.bin(x[j]);
            if (b >= lo_bin && b <= hi_bin) atomicAdd(&s->wide[(chi - comp) >> shift], by_mass ? r.weight(x[j]) : 1ull);
        }
    });
    pick_total(r, s->wide, s->wide_tot);
    u64 in_bin[PER], all = 0ull;  // a thread's bins lie side by side
#pragma unroll
    for (int i = 0; i < PER; i++) all += in_bin[i] = s->wide_tot[PER * tid + i];
    u64 c = up + pick_scan(all, s->red) - all;
#pragma unroll
    for (int i = 0; i < PER; i++) {  // one bin of all, or none
        if ((double)c < target && (double)(c + in_bin[i]) >= target) s->b1 = PER * tid + i;
        c += in_bin[i];
    }
    __syncthreads();
    const int last = (int)((chi - clo) >> shift), b = min(s->b1, last);
    const u64 top = chi - ((u64)b << shift);
    *chi_p = top;
    if (b < last) *clo_p = top - ((1ull << shift) - 1ull);
}

// Where the prefix of {comp >= tau0} ends whose metric (number of tokens, or mass) first reaches `target`:
// the comp of its last token. s->hist holds this CTA's histogram of the bins: tokens, or for a mass their
// weights over that of the bin's middle, in units of 1 / unit. Those bound the metric: the border lies in one bin or
// in a few, whose tokens are the members. While they are too many, their range of comps is split into bins of
// exact sums: the border lies in one of them. A range starts and ends with a member and holds 512 comps or more, so
// each time at least two bins are occupied, and what is left is smaller by a factor of 512: seven times at most, the
// comps having 64 bits.
// *kept: the metric that this warp's tokens have in the prefix.
__device__ u64 pick_border(PickRow& r, bool by_mass, double target, double unit, u64 tau0, u64* kept) {
    PickShared* s = r.s;
    const int tid = threadIdx.x;
    u64 chi = ~0ull, clo = 0ull;  // the members' range
    u64 up = 0ull;                // metric of what lies above them
    if (tid == 0) s->b1 = s->b2 = kPickBins;
    pick_total(r, s->hist, s->tot);
    // bounds of the metric up to each bin; a thread's bins lie side by side
    const double per_unit = kOne / unit, e = 0.52 / unit + 1.1e-5;
    double lo[kPickPer], hi[kPickPer], lo_all = 0.0, hi_all = 0.0;
#pragma unroll
    for (int i = 0; i < kPickPer; i++) {
        const int b = kPickPer * tid + i;
        const double n = (double)s->tot[b];
        lo[i] = hi[i] = n;
        if (by_mass && n > 0.0) {
            // a token's share is rounded by half a unit and lies above 0.99; 1e-5: the fp32 places and shares;
            // 1e-6: the power here
            const double top = n * per_unit * (double)pick_ex2(-kPickSpan / kPickBins * (float)b);
            hi[i] = top * (1.0 + e);
            lo[i] = top * (1.0 - e);
        }
        lo_all += lo[i];
        hi_all += hi[i];
    }
    double* red = reinterpret_cast<double*>(s->red);
    double cl = pick_scan(lo_all, red) - lo_all, ch = pick_scan(hi_all, red) - hi_all;
    // sums of doubles may be off by a few parts in 2^53 per bin
    const double early = target * (1.0 - 1e-12), late = by_mass ? target * (1.0 + 1e-12) : target;
    // the first bins that reach the target; threads well behind them stay out
    bool no1 = ch > early * (1.0 + 1e-9), no2 = cl > late * (1.0 + 1e-9);
#pragma unroll
    for (int i = 0; i < kPickPer; i++) {
        ch += hi[i];
        cl += lo[i];
        if (!no1 && ch >= early) {
            atomicMin(&s->b1, kPickPer * tid + i);
            no1 = true;
        }
        if (!no2 && cl >= late) {
            atomicMin(&s->b2, kPickPer * tid + i);
            no2 = true;
        }
    }
    if (tid == 0 && !(early > 0.0)) atomicMin(&s->b1, 0);
    if (tid == 0 && !(late > 0.0)) atomicMin(&s->b2, 0);
    __syncthreads();
    if (!by_mass && s->b1 == kPickBins) {  // fewer tokens than that: all of them
        *kept = 0ull;                      // (only the kept mass is asked for)
        return tau0;
    }
    const int lo_bin = min(s->b1, kPickBins - 1), hi_bin = min(max(s->b2, s->b1), kPickBins - 1);
    while (true) {
        if (tid == 0) s->count = 0u;
        __syncthreads();
        // what lies above the members, exactly; the members themselves, and their range
        u64 first = ~0ull, last = 0ull;
        up = 0ull;
        // weights are dear: the warp gathers the tokens that lie above, and weighs them four a lane
        float* gather = reinterpret_cast<float*>(s->pair) + (tid >> 5) * kPickGather;
        int held = 0;
        const int lane = tid & 31;
        auto weigh = [&] {
            __syncwarp();
            double w = 0.0;
#pragma unroll
            for (int j = 0; j < kPickGather / 32; j++) w += lane + 32 * j < held ? r.mass(gather[lane + 32 * j]) : 0.0;
            up += (u64)w;
            __syncwarp();
            held = 0;
        };
        r.each([&](const float (&x)[4], const int (&idx)[4], const bool (&is)[4]) {
            bool over[4], in[4], some = false, members = false;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int b = is[j] ? r.bin(x[j]) : kPickBins;
                over[j] = b < lo_bin;
                in[j] = b >= lo_bin && b <= hi_bin;
                some |= over[j];
                members |= in[j];
            }
            if (tau0 != 0ull && __any_sync(0xffffffffu, some)) {
#pragma unroll
                for (int j = 0; j < 4; j++) over[j] = over[j] && pick_comp(x[j], idx[j]) >= tau0;
            }
            if (__any_sync(0xffffffffu, members)) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const u64 comp = pick_comp(x[j], idx[j]);
                    if (in[j]) {
                        over[j] = comp > chi && comp >= tau0;
                        in[j] = comp <= chi && comp >= clo && comp >= tau0;
                        some |= over[j];
                    }
                    if (in[j]) {
                        first = pick_min(first, comp);
                        last = pick_max(last, comp);
                    }
                    pick_append(s, in[j], comp);
                }
            }
            if (!__any_sync(0xffffffffu, some)) return;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (!by_mass) {
                    up += over[j];
                    continue;
                }
                const unsigned m = __ballot_sync(0xffffffffu, over[j]);
                if (held + __popc(m) > kPickGather) weigh();
                if (over[j]) gather[held + __popc(m & ((1u << lane) - 1u))] = x[j];
                held += __popc(m);
            }
        });
        if (held) weigh();
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) up += __shfl_xor_sync(0xffffffffu, up, o);
        const u64 warp_up = up;
        up = pick_sum(r, (tid & 31) == 0 ? up : 0ull);
        const int total = pick_collect(r, r.exchange(s->count), 1, kPickRank);
        if (total >= 0) {
            if (r.rank == 0) {
                // the token up to which the running metric reaches the target: first its key, by bisection, then its
                // place among equal ones
                const u64 mine = tid < total ? s->list[tid] : 0ull;
                const uint32_t key = (uint32_t)(mine >> 32);
                const u64 own = tid < total ? (by_mass ? r.weight(pick_value(mine)) : 1ull) : 0ull;
                const uint32_t low_key = (uint32_t)pick_reduce(tid < total ? (u64)key : ~0ull, s->red, pick_min);
                const uint32_t top_key = (uint32_t)pick_reduce((u64)key, s->red, pick_max);
                auto reach = [&](uint32_t k) { return up + pick_reduce(key >= k ? own : 0ull, s->red, pick_add); };
                uint32_t lo_key = low_key;
                if ((double)up >= target) {
                    lo_key = top_key;
                } else if ((double)reach(low_key) >= target) {
                    // digit by digit: sums of the weights (below 2^43) by digit in two words of 22 and 21 bits
                    uint32_t* words = reinterpret_cast<uint32_t*>(s->pair);
                    u64 over = up;
                    const uint32_t off = key - low_key;
                    uint32_t prefix = 0u;
                    for (int bit = 32 - __clz((int)(top_key - low_key)); bit > 0;) {
                        const int next = max(0, bit - kPickDigit);
                        words[tid] = words[kPickThreads + tid] = 0u;
                        __syncthreads();
                        if (own && (bit == 32 || off >> bit == prefix)) {
                            const uint32_t d = (off >> next) & ((1u << (bit - next)) - 1u);
                            atomicAdd(&words[d], (uint32_t)own & 0x3FFFFFu);
                            atomicAdd(&words[kPickThreads + d], (uint32_t)(own >> 22));
                        }
                        __syncthreads();
                        const int d = kPickThreads - 1 - tid;  // larger keys first
                        const u64 n = words[d] + ((u64)words[kPickThreads + d] << 22), upto = over + pick_scan(n, s->red);
                        if ((double)upto >= target && (double)(upto - n) < target) {
                            s->b1 = d;
                            s->border = upto - n;
                        }
                        __syncthreads();
                        over = s->border;
                        prefix = prefix << (bit - next) | (uint32_t)s->b1;
                        bit = next;
                    }
                    lo_key = low_key + prefix;
                }
                const u64 over = lo_key < top_key ? reach(lo_key + 1u) : up;
                const bool equal = tid < total && key == lo_key;
                const int equals = __syncthreads_count(equal);
                if (tid == 0) s->tau = tau0;  // no token at all
                s->pair[tid] = make_ulonglong2(equal ? mine : 0ull, 0ull);
                __syncthreads();
                if (equal) {
                    u64 at = 0ull;  // equal ones of lower index
                    if (equals > 1)
                        for (int j = 0; j < total; j++) at += s->pair[j].x > mine;
                    // the first whose sum reaches the target; the last if none does
                    const bool before = at > 0ull && (double)(over + at * own) >= target;
                    if (!before && ((double)(over + (at + 1ull) * own) >= target || (int)at == equals - 1)) s->tau = mine;
                }
                __syncthreads();
                if (tid > 0 && tid < r.C) cg::this_cluster().map_shared_rank(s, tid)->tau = s->tau;
            }
            r.sync();
            const u64 tau = s->tau;
            u64 mine = 0ull;  // this CTA's members lie first in its list
            for (int i = tid & 31; i < (int)s->count; i += 32) {
                const u64 comp = s->list[i];
                const int idx = pick_index(comp);
                if (comp >= tau && idx >= r.w0 && idx < r.w1) mine += by_mass ? r.weight(pick_value(comp)) : 1ull;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
            *kept = warp_up + mine;
            return tau;
        }
        // too many: split the members' range of comps
        first = pick_reduce(first, s->red, pick_min);
        last = pick_reduce(last, s->red, pick_max);
        const u64* x0 = r.exchange(first);
        for (int i = 0; i < r.C; i++) first = pick_min(first, x0[i]);
        const u64* x1 = r.exchange(last);
        for (int i = 0; i < r.C; i++) last = pick_max(last, x1[i]);
        clo = first;
        chi = last;
        pick_split(r, by_mass, target, tau0, lo_bin, hi_bin, up, &clo, &chi);
    }
}

__device__ __forceinline__ void pick_write(const PickArgs& a, int row, int id, float p) {
    a.ids[row] = id;
    if (a.probs) a.probs[row] = p;
}

// CTA 0 of the row ends it: `n` tokens in s->list, in index order, that hold the kept set; `rest` is the mass of
// the others. False if the top-p border lies among those.
__device__ bool pick_short(const PickArgs& a, PickRow& r, int row, int n, int K, float P, double mp, u64 rest) {
    PickShared* s = r.s;
    const int tid = threadIdx.x;
    const u64* list = s->list;
    u64 low = ~0ull;
    for (int i = tid; i < n; i += kPickThreads) low = pick_min(low, list[i] >> 32);
    const uint32_t least = (uint32_t)pick_reduce(low, s->red, pick_min);
    const uint32_t most = f32_order_key(r.mx);
    auto count = [&](uint32_t key) {  // tokens of keys at least `key`
        int c = 0;
        if (n <= kPickThreads) return __syncthreads_count(tid < n && (uint32_t)(s->list[tid] >> 32) >= key);
        for (int i = tid; i < n; i += kPickThreads) c += (uint32_t)(s->list[i] >> 32) >= key;
        return (int)pick_reduce((u64)c, s->red, pick_add);
    };
    auto mass = [&](uint32_t key) {
        u64 m = 0ull;
        for (int i = tid; i < n; i += kPickThreads)
            if ((uint32_t)(list[i] >> 32) >= key) m += r.weight(pick_value(list[i]));
        return pick_reduce(m, s->red, pick_add);
    };
    // kept: keys above tau, and the first `ties` (by index) equal to it
    uint32_t tau = least;
    u64 ties = ~0ull;
    if (K < n) {
        uint32_t lo = least, hi = most;  // the largest key that K tokens reach
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo + 1u) / 2u;
            if (count(mid) >= K)
                lo = mid;
            else
                hi = mid - 1u;
        }
        tau = lo;
        ties = (u64)(K - (tau < most ? count(tau + 1u) : 0));
    }
    if (K < n && K <= kPickTopK) {  // on with the top-k alone, in index order
        const int per = (n + kPickThreads - 1) / kPickThreads, i0 = min(n, tid * per), i1 = min(n, i0 + per);
        u64 both = 0ull;  // keys above tau, keys equal to it
        for (int i = i0; i < i1; i++) {
            const uint32_t k = (uint32_t)(list[i] >> 32);
            both += ((u64)(k > tau) << 32) + (k == tau);
        }
        const u64 before = pick_scan(both, s->red) - both;
        uint32_t above = (uint32_t)(before >> 32), equal = (uint32_t)before;
        for (int i = i0; i < i1; i++) {
            const uint32_t k = (uint32_t)(list[i] >> 32);
            if (k > tau || (k == tau && equal < ties)) s->top[above + min((u64)equal, ties)] = list[i];
            above += k > tau;
            equal += k == tau;
        }
        __syncthreads();
        list = s->top;
        n = K;
        ties = ~0ull;
    }
    u64 bar = 0ull;  // comps from here on, as far as decided below
    if (P < 1.0f && n <= kPickPairs) {
        // the mass in front of each token, over all pairs
        const u64 mine = tid < n ? list[tid] : 0ull, own = tid < n ? r.weight(pick_value(mine)) : 0ull;
        s->pair[tid] = make_ulonglong2(mine, own);
        const u64 M = pick_reduce(own, s->red, pick_add);
        const double need = (double)P * (double)(M + rest);
        if ((double)M < need) return false;
        u64 front = 0ull;
        if (tid < n)
#pragma unroll 8
            for (int j = 0; j < n; j++) {
                const ulonglong2 q = s->pair[j];
                front += q.x > mine ? q.y : 0ull;
            }
        bar = pick_reduce(tid < n && (front == 0ull || (double)front < need) ? mine : ~0ull, s->red, pick_min);
        tau = 0u;
    } else if (P < 1.0f) {
        const u64 wt = r.weight(pick_value((u64)tau << 32)), over = tau < most ? mass(tau + 1u) : 0ull;
        const u64 M = (ties == ~0ull ? mass(tau) : over + ties * wt) + rest;
        const double need = (double)P * (double)M;
        // the largest key above tau down to which the mass reaches `need`; else tau
        if (tau < most && (double)over >= need) {
            uint32_t lo = tau + 1u, hi = most;
            while (lo < hi) {
                const uint32_t mid = lo + (hi - lo + 1u) / 2u;
                if ((double)mass(mid) >= need)
                    lo = mid;
                else
                    hi = mid - 1u;
            }
            tau = lo;
            ties = ~0ull;
        } else if ((double)(M - rest) < need) {
            return false;
        }
        const u64 w = r.weight(pick_value((u64)tau << 32)), above = tau < most ? mass(tau + 1u) : 0ull;
        u64 m = w ? (u64)fmax(0.0, (need - (double)above) / (double)w) : 1ull;
        m = m > 1ull ? m - 1ull : 1ull;
        while (m < ties && m < (u64)n && (double)(above + m * w) < need) m++;
        ties = pick_min(ties, m);
    }
    // sums of the kept weights in index order; a thread's tokens lie side by side
    const int per = (n + kPickThreads - 1) / kPickThreads, i0 = min(n, tid * per), i1 = min(n, i0 + per);
    u64 seen0 = 0ull;
    if (ties != ~0ull) {
        u64 equal = 0ull;
        for (int i = i0; i < i1; i++) equal += (uint32_t)(list[i] >> 32) == tau;
        seen0 = pick_scan(equal, s->red) - equal;
    }
    auto kept = [&](int i, u64& seen) -> u64 {
        const u64 c = list[i];
        const uint32_t k = (uint32_t)(c >> 32);
        if (k < tau || c < bar || (k == tau && seen++ >= ties)) return 0ull;
        const u64 w = r.weight(pick_value(c));
        return (double)w >= mp * kOne ? w : 0ull;
    };
    u64 sum = 0ull, seen = seen0;
    for (int i = i0; i < i1; i++) sum += kept(i, seen);
    u64 run = pick_scan(sum, s->red);
    const u64 S = pick_reduce(run, s->red, pick_max);
    run -= sum;
    // the first token whose running sum passes the target; the last kept one if none does
    const double target = (double)a.u[row] * (double)S;
    const bool inside = !((double)run > target) && ((double)(run + sum) > target || run + sum == S);
    if (sum > 0ull && (inside || (run == 0ull && (double)run > target))) {
        u64 got = 0ull;
        int id = -1;
        seen = seen0;
        for (int i = i0; i < i1; i++) {
            const u64 w = kept(i, seen);
            if (w == 0ull) continue;
            run += w;
            got = w;
            id = pick_index(list[i]);
            if ((double)run > target) break;
        }
        pick_write(a, row, id, (float)((double)got / (double)S));
    }
    return true;
}

__global__ void __launch_bounds__(kPickThreads, 2) pick_kernel(PickArgs a, int C, int chunk) {
    extern __shared__ __align__(16) unsigned char pick_sm[];
    PickShared* s = reinterpret_cast<PickShared*>(pick_sm);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / C, V = a.V;
    PickRow r;
    r.s = s;
    r.C = C;
    r.rank = blockIdx.x - row * C;
    r.turn = 0;
    r.endless = false;
    r.l = a.logits + (size_t)row * a.ld;
    r.V = V;
    r.vec = ((uintptr_t)r.l & 15) == 0;
    r.v0 = min(V, r.rank * chunk);
    r.v1 = min(V, r.v0 + chunk);
    const int seg = (r.v1 - r.v0 + kPickWarps * 128 - 1) / (kPickWarps * 128) * 128;
    r.w0 = min(r.v1, r.v0 + warp * seg);
    r.w1 = min(r.v1, r.w0 + seg);
    const float Tf = a.temperature ? a.temperature[row] : 1.0f;
    const int K = a.top_k ? a.top_k[row] : 0;
    const float P = a.top_p ? a.top_p[row] : 1.0f;
    const float mf = a.min_p ? a.min_p[row] : 0.0f;
    const double mp = mf > 0.0f ? fmin((double)mf, 1.0) : 0.0;  // NaN: off
    if (tid < 64) s->pow2[tid] = exp2((double)tid / 64.0);
    if (tid == 0) s->count = 0u;

    // maxima: of each lane's four columns, and the first index of the row's
    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, best = -INFINITY;
    int at = 0;
#pragma unroll 4
    for (int i = r.w0; i < r.w1; i += 128) {
        float x[4];
        r.load(i + 4 * lane, x);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            m4[j] = fmaxf(m4[j], x[j]);
            if (x[j] > best) {
                best = x[j];
                at = i + 4 * lane + j;
            }
        }
    }
    u64 top = best > -INFINITY ? pick_comp(best, at) : 0ull;
    top = pick_reduce(top, s->red, pick_max);
    if (C > 1) {
        // Another CTA's shared memory exists once that CTA has started: here each leaves its maximum in its own, and
        // takes the others' behind the barrier.
        if (tid == 0) s->x[r.turn][r.rank] = top;
        r.sync();
        top = lane < C ? r.of(lane)->x[r.turn][lane] : 0ull;
#pragma unroll
        for (int o = kPickMaxCluster / 2; o > 0; o >>= 1) top = pick_max(top, __shfl_xor_sync(0xffffffffu, top, o));
        top = __shfl_sync(0xffffffffu, top, 0);
    }
    if (top == 0ull || !(Tf > 0.0f)) {
        if (r.rank == 0 && tid == 0) pick_write(a, row, top ? pick_index(top) : -1, top ? 1.0f : 0.0f);
        r.sync();  // until the others have read
        return;
    }
    r.mx = pick_value(top);
    r.endless = isinf(r.mx);
    if (r.endless) {
        r.mx = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) m4[j] = r.seen(m4[j]);
    }
    r.c = 1.44269504088896340736 / (double)Tf;
    // Bins of a difference of 1. fp32 holds it for T above 7e-29; below, 2^-64 of it, the logits times 2^64. Where the
    // maximum is too large for that, every other logit is 2^-84 away or more: 1e30 puts it behind all bins too. A
    // difference passes fp32's range only under a maximum above 2^103: there of halves.
    const double per_one = r.c * (kPickBins / (double)kPickSpan);
    r.lift = r.mx >= 0x1p100f ? 0.5f : per_one > 1e30 && fabsf(r.mx) < 0x1p-60f ? 0x1p64f : 1.0f;
    r.mx_lift = r.mx * r.lift;
    r.bin_scale = (float)fmin(per_one / r.lift, 1e30);

    r.pooled = -1;
    const bool by_k = K > 0 && K < V, by_p = P < 1.0f;
    // the last bin whose tokens go to the pools (-1: no pools)
    int most = -1;
    const bool bound_k = by_k && K <= kPickTopK;
    if (by_p && !by_k) {
        // all tokens below 2^-e weigh less than 2^-e V, which is less than (1 - P) of all when 2^e = V / ((1 - P) M')
        // for a part M' of the mass; here that of the maxima, rounded down
        float part = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (m4[j] > -INFINITY) part += exp2f(-kPickSpan / kPickBins * r.place(m4[j]));
        const double M = fmax(1.0, 0.99 / kOne * (double)pick_sum(r, (u64)(part * (float)kOne)));
        const double e = log2((double)V / ((1.0 - (double)P) * M));
        most = max(0, min(kPickBins - 1, (int)(e * (kPickBins / (double)kPickSpan)) + 1));
    } else if (bound_k) {
        // K of the CTA's maxima: at least K logits are as large
        for (int b = tid; b < kPickBins; b += kPickThreads) s->hist[b] = 0u;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (m4[j] > -INFINITY) atomicAdd(&s->hist[r.bin(m4[j])], 1u);
        if (tid == 0) s->b1 = kPickBins - 1;
        __syncthreads();
        u64 in_bin[kPickPer], here = 0ull;
#pragma unroll
        for (int i = 0; i < kPickPer; i++) here += in_bin[i] = s->hist[kPickPer * tid + i];
        u64 c = pick_scan(here, s->red) - here;
#pragma unroll
        for (int i = 0; i < kPickPer; i++) {
            if (c < (u64)K && c + in_bin[i] >= (u64)K) s->b1 = kPickPer * tid + i;  // one bin of all
            c += in_bin[i];
        }
        __syncthreads();
        u64 b = s->b1;
        const u64* e = r.exchange(b);
        for (int i = 0; i < C; i++) b = pick_min(b, e[i]);
        most = (int)b;
    } else if (!by_k && mp > 0x1p-38) {
        most = min(kPickBins - 1, (int)(-log2(mp) * (kPickBins / (double)kPickSpan) * (1.0 + 1e-5)) + 1);
    }
    const double unit = (double)(1u << (V <= 1 << 17 ? 14 : 11));  // V of them fit 32 bits
    u64 rest = 0ull, M = 0ull;
    bool have = false;
    if (most >= 0) {
        // tokens of bins up to `most` into the warp's pool, in index order; the others' mass for top-p
        int n = 0;
        const bool sums = by_p && !by_k;
        const float limit = most < kPickBins - 1 ? (float)most + 0.5f : INFINITY;  // bin <= most: up to it
        double others = 0.0, all = 0.0;
        if (sums) {
            for (int b = tid; b < kPickBins; b += kPickThreads) s->hist[b] = 0u;
            __syncthreads();
        }
        float ahead[4];
        if (r.w0 < r.w1) r.load(r.w0 + 4 * lane, ahead);
        for (int i = r.w0; i < r.w1; i += 128) {
            const float q[4] = {ahead[0], ahead[1], ahead[2], ahead[3]};
            if (i + 128 < r.w1) r.load(i + 128 + 4 * lane, ahead);
            float place[4];
            bool in[4];
            unsigned own = 0u;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                place[j] = r.place(q[j]);
                in[j] = q[j] > -INFINITY && !(place[j] > limit);
                own += in[j];
            }
            if (sums) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const double w = r.mass(q[j]);
                    all += w;
                    others += in[j] ? 0.0 : w;
                }
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (in[j]) r.share(place[j], (float)unit);
            }
            if (!__any_sync(0xffffffffu, own != 0u)) continue;
            unsigned at = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned y = __shfl_up_sync(0xffffffffu, at, o);
                if (lane >= o) at += y;
            }
            const int total = __shfl_sync(0xffffffffu, at, 31);
            at += n - own;
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (in[j]) {
                    if (at < kPickPool) s->pool[warp][at] = (uint16_t)(i + 4 * lane + j - r.w0);
                    at++;
                }
            n += total;
        }
        rest = (u64)others;
        M = (u64)all;
        // all of them to CTA 0, when they are few
        if (lane == 0) s->inside[warp] = (uint32_t)n;
        __syncthreads();
        uint32_t before = 0u, total = 0u, largest = 0u;
        for (int i = 0; i < kPickWarps; i++) {
            const uint32_t c = s->inside[i];
            if (i < warp) before += c;
            total += c;
            largest = max(largest, c);
        }
        const bool fits = largest <= kPickPool && total <= kPickList;
        if (fits)
            for (int i = lane; i < n; i += 32) {
                const int idx = r.w0 + s->pool[warp][i];
                s->list[before + i] = pick_comp(r.at(idx), idx);
            }
        __syncthreads();
        // the CTAs' sums, numbers of tokens and largest pools, in one exchange
        if (sums) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                rest += __shfl_xor_sync(0xffffffffu, rest, o);
                M += __shfl_xor_sync(0xffffffffu, M, o);
            }
            if (lane == 0) {
                s->red[warp] = rest;
                s->red2[warp] = M;
            }
            __syncthreads();
            rest = M = 0ull;
            for (int w = 0; w < kPickWarps; w++) {
                rest += s->red[w];
                M += s->red2[w];
            }
        }
        if (tid < 4 * C)
            r.of(tid >> 2)->x4[r.rank][tid & 3] = (tid & 2) == 0 ? ((tid & 1) == 0 ? rest : M)
                                                  : (tid & 1) == 0 ? (u64)(fits ? total : kPickList + 1u) : (u64)largest;
        r.sync();
        rest = M = 0ull;
        u64 widest = 0ull;
        for (int i = 0; i < C; i++) {
            rest += s->x4[i][0];
            M += s->x4[i][1];
            widest = pick_max(widest, s->x4[i][3]);
        }
        // the border is among the histogram's tokens: it serves the passes below
        have = sums && (double)P * (double)M <= (double)(M - rest);
        const int found = pick_collect(r, &s->x4[0][2], 4, kPickList);
        if (found >= 0) {
            bool done = true;
            if (r.rank == 0) done = pick_short(a, r, row, found, by_k ? K : found, P, mp, rest);
            if (!sums) return;
            const u64* e = r.exchange(done ? 1ull : 0ull);
            if (e[0]) return;
        } else {
            // pools that are too many for one CTA serve the passes below
            if (widest <= (u64)kPickPool) r.pooled = n;
        }
    }

    u64 tau = 0ull, sum = 0ull;
    for (int pass = by_k ? 0 : 1; pass < (by_p ? 2 : 1); pass++) {
        if (!have) {
            // histogram of the bins among {comp >= tau}: tokens, or for top-p their weights, and the mass
            if (pass == 1 && !by_k) r.pooled = -1;  // the pools miss the border
            for (int b = tid; b < kPickBins; b += kPickThreads) s->hist[b] = 0u;
            __syncthreads();
            double all = 0.0;
            r.each([&](const float (&x)[4], const int (&idx)[4], const bool (&is)[4]) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const bool in = is[j] && (tau == 0ull || pick_comp(x[j], idx[j]) >= tau);
                    if (pass == 1) {
                        const double w = r.mass(x[j]);
                        all += in ? w : 0.0;
                        if (in) r.share(r.place(x[j]), (float)unit);
                    } else if (in) {
                        atomicAdd(&s->hist[r.bin(x[j])], 1u);
                    }
                }
            });
            if (pass == 1) M = pick_sum(r, (u64)all);
        }
        tau = pick_border(r, pass == 1, pass == 1 ? (double)P * (double)M : (double)K, unit, tau, &sum);
    }

    // sums of the kept weights by warp, in index order
    auto kept = [&](float q, int i) -> u64 {
        if (!(q > -INFINITY) || (tau != 0ull && pick_comp(q, i) < tau)) return 0ull;
        const u64 w = r.weight(q);
        return (double)w >= mp * kOne ? w : 0ull;
    };
    if (!by_p || mp > 0.0) {  // else the border's search has summed them
        double all = 0.0;     // whole numbers up to 2^53: a lane has 2^11 of them at most
        r.each([&](const float (&x)[4], const int (&idx)[4], const bool (&is)[4]) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const double w = r.mass(x[j]);
                all += is[j] && w >= mp * kOne && (tau == 0ull || pick_comp(x[j], idx[j]) >= tau) ? w : 0.0;
            }
        });
        sum = (u64)all;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (lane < C) (C > 1 ? cg::this_cluster().map_shared_rank(s, lane) : s)->sums[r.rank][warp] = sum;
    r.sync();
    u64 before = 0ull, S = 0ull;
    for (int i = 0; i < C * kPickWarps; i++) {
        const u64 v = s->sums[i / kPickWarps][i % kPickWarps];
        if (i < r.rank * kPickWarps + warp) before += v;
        S += v;
    }
    // the first token whose running sum passes the target; the last kept one if none does
    const double target = (double)a.u[row] * (double)S;
    const bool inside = !((double)before > target) && ((double)(before + sum) > target || before + sum == S);
    if (sum == 0ull || !(inside || (before == 0ull && (double)before > target))) return;
    int id = -1;
    u64 got = 0ull;
    const bool pools = r.pooled >= 0;
    const int end = pools ? r.pooled : r.w1;
    for (int i = pools ? 0 : r.w0; i < end; i += 128) {
        float q[4];
        int idx[4];
        if (pools) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int k = i + 4 * lane + j;
                idx[j] = k < end ? r.w0 + s->pool[warp][k] : -1;
            }
#pragma unroll
            for (int j = 0; j < 4; j++) q[j] = idx[j] >= 0 ? r.at(idx[j]) : -INFINITY;
        } else {
            r.load(i + 4 * lane, q);
#pragma unroll
            for (int j = 0; j < 4; j++) idx[j] = i + 4 * lane + j;
        }
        u64 w[4], own = 0ull;
#pragma unroll
        for (int j = 0; j < 4; j++) own += w[j] = kept(q[j], idx[j]);
        u64 incl = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        u64 run = before + incl - own;
        // this lane's last kept token up to the one that passes the target
        int mine = -1;
        u64 mw = 0ull;
        bool passed = false;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (w[j] == 0ull || passed) continue;
            run += w[j];
            mine = idx[j];
            mw = w[j];
            passed = (double)run > target;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, passed), any = __ballot_sync(0xffffffffu, mine >= 0);
        if (any) {
            const int src = hit ? __ffs(hit) - 1 : 31 - __clz(any);
            id = __shfl_sync(0xffffffffu, mine, src);
            got = __shfl_sync(0xffffffffu, mw, src);
        }
        if (hit) break;
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) pick_write(a, row, id, (float)((double)got / (double)S));
}

}  // namespace

// CTAs of a row: up to 4 CTAs per SM in all, while a CTA keeps 4096 logits or
// more. Two are resident; rows differ in their work, so a second wave evens it
// out (256 mixed rows of 128256: 357 us with one CTA each, 250 with two, 241
// with four; 140 rows of top-p alone with two, four and eight: 207, 183 and 271).
// 64 rows would rather have one wave (top-p alone with two, four and eight each: 195,
// 128 and 134 us; mixed: 126, 83 and 116). Below 4096 logits the exchanges cost more
// than the passes (62 rows of 14783, k = 1150: 35 us, 40 at 2048).
int launch_pick(const PickArgs& a, cudaStream_t s) {
    if (a.rows == 0) return JYC_OK;
    const int sms = sm_count();
    if (sms == 0) return cuda_fail(cudaErrorNoDevice, "sample_batch: device query");
    int C = 1;
    while (C < kPickMaxCluster && (long long)a.rows * 2 * C <= 4 * sms && a.V / (2 * C) >= 4096) C *= 2;
    const int chunk = ((a.V + C - 1) / C + 3) / 4 * 4;
    if (int e = max_dynamic_smem(reinterpret_cast<const void*>(pick_kernel), (int)sizeof(PickShared))) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(a.rows * C));
    cfg.blockDim = dim3(kPickThreads);
    cfg.dynamicSmemBytes = sizeof(PickShared);
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)C;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    JYC_CUDA(cudaLaunchKernelEx(&cfg, pick_kernel, a, C, chunk));
    JYC_LAUNCHED();
    return JYC_OK;
}

}  // namespace jyc
