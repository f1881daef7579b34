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
// shared memory, so one launch serves one row or hundreds:
//   greedy   the maximum, one pass.
//   top-k up to 1024   every lane keeps four maxima of its part; the k-th
//            largest of a CTA's maxima bounds the k-th largest logit from
//            below, and the few tokens above the bound are sorted by one CTA,
//            which ends the row alone.
//   otherwise  a histogram of counts over (max - l) / T, whose bins bound the
//            mass above them; the tokens of the bins where the border may lie
//            are sorted (or split again while they are too many), then the
//            kept weights are summed in index order.
// Floor: one read of the logits. Later passes find them in L2.
#include <cooperative_groups.h>

#include <algorithm>

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace jyc {

namespace {

typedef unsigned long long u64;

constexpr int kPickThreads = 512, kPickWarps = kPickThreads / 32;
constexpr int kPickList = 4096;      // tokens that one CTA sorts
constexpr int kPickTopK = 1024;      // largest k of the short way
constexpr int kPickBins = 1024;
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

struct PickShared {
    u64 list[kPickList];
    u64 w[kPickTopK];
    uint32_t hist[kPickBins], tot[kPickBins];
    double pow2[64];                   // 2^(j / 64)
    u64 x[2][kPickMaxCluster];         // exchanges between CTAs, two turns
    u64 sums[kPickMaxCluster][kPickWarps];
    u64 red[kPickWarps];
    u64 tau;
    uint32_t count;
    int b1, b2;
};

// One row, as a CTA sees it.
struct PickRow {
    const float* l;
    int V, v0, v1, w0, w1;  // the CTA's part, the warp's part
    bool vec;
    float mx;
    double c;               // log2(e) / T
    float bin_scale;
    int C, rank, turn;
    PickShared* s;

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
    }
    // 2^t by 2^(j / 64) and the exponential series: |s| <= ln 2 / 128, remainder s^5 / 120 < 4e-14
    __device__ __forceinline__ u64 weight(float x) const {
        if (x == mx) return (u64)kOne;
        const double t = ((double)x - (double)mx) * c;
        if (!(t >= -40.0)) return 0ull;  // NaN and -inf too
        const double m = __fma_rn(t, 64.0, 0x1.8p52);
        const int n = __double2loint(m);
        const double s1 = __fma_rn(m - 0x1.8p52, -1.0 / 64.0, t) * 0.693147180559945309417;
        double p = __fma_rn(s1, 1.0 / 24.0, 1.0 / 6.0);
        p = __fma_rn(p, s1, 0.5);
        p = __fma_rn(p, s1, 1.0);
        p = __fma_rn(p, s1, 1.0) * s->pow2[n & 63];
        const double q = __hiloint2double(__double2hiint(p) + (((n >> 6) + 42) << 20), __double2loint(p));
        return (u64)__double_as_longlong(q + 0x1p52) & 0xFFFFFFFFFFFFFull;
    }
    // bin of a logit above -inf: larger logits never lie in a later bin
    __device__ __forceinline__ int bin(float x) const {
        if (x == mx) return 0;
        const float b = __fmul_rn(__fsub_rn(mx, x), bin_scale);
        return b < (float)(kPickBins - 1) ? (int)b : kPickBins - 1;
    }
    __device__ void sync() const {
        if (C > 1)
            cg::this_cluster().sync();
        else
            __syncthreads();
    }
    // v of every CTA, in s->x[turn][rank of it] after the call; v from thread 0
    __device__ const u64* exchange(u64 v) {
        turn ^= 1;
        if (C > 1) {
            if (threadIdx.x == 0)
                for (int r = 0; r < C; r++) cg::this_cluster().map_shared_rank(s, r)->x[turn][rank] = v;
        } else if (threadIdx.x == 0) {
            s->x[turn][0] = v;
        }
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

// bitonic sort, descending; n a power of two
__device__ void pick_sort(u64* a, int n) {
    __syncthreads();
    for (int k = 2; k <= n; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int i = threadIdx.x; i < n / 2; i += kPickThreads) {
                const int lo = (i & ~(j - 1)) * 2 + (i & (j - 1)), hi = lo + j;
                const u64 x = a[lo], y = a[hi];
                if ((x < y) == ((lo & k) == 0)) {
                    a[lo] = y;
                    a[hi] = x;
                }
            }
            __syncthreads();
        }
}
__device__ __forceinline__ int pick_pow2(int n) { return n <= 1 ? 1 : 1 << (32 - __clz(n - 1)); }

// Appends comp to the CTA's list where `take` holds (whole warps call it); s->count counts on past the end.
__device__ __forceinline__ void pick_append(PickShared* s, bool take, u64 comp) {
    const unsigned m = __ballot_sync(0xffffffffu, take);
    if (m == 0u) return;
    const int lane = threadIdx.x & 31;
    uint32_t at = 0u;
    if (lane == 0) at = atomicAdd(&s->count, (uint32_t)__popc(m));
    at = __shfl_sync(0xffffffffu, at, 0) + __popc(m & ((1u << lane) - 1u));
    if (take && at < kPickList) s->list[at] = comp;
}

// The CTAs' lists joined in the first one's, when they fit. Returns their total (-1: too many), the same in
// every CTA; the list is complete in CTA 0 after the next sync.
__device__ int pick_collect(PickRow& r) {
    __syncthreads();
    const uint32_t mine = r.s->count;
    const u64* x = r.exchange(mine);
    u64 total = 0ull, before = 0ull;
    for (int i = 0; i < r.C; i++) {
        if (i < r.rank) before += x[i];
        total += x[i];
    }
    if (total > (u64)kPickList) return -1;
    if (r.rank > 0) {
        u64* to = cg::this_cluster().map_shared_rank(r.s, 0)->list;
        for (uint32_t i = threadIdx.x; i < mine; i += kPickThreads) to[before + i] = r.s->list[i];
    }
    return (int)total;
}

// Sums of the CTA's histograms in s->tot of every CTA.
__device__ void pick_total(PickRow& r) {
    r.sync();
    if (r.C == 1) {
        for (int b = threadIdx.x; b < kPickBins; b += kPickThreads) r.s->tot[b] = r.s->hist[b];
        __syncthreads();
        return;
    }
    const int per = kPickBins / r.C;
    for (int i = threadIdx.x; i < per; i += kPickThreads) {
        const int b = r.rank * per + i;
        uint32_t n = 0u;
        for (int c = 0; c < r.C; c++) n += cg::this_cluster().map_shared_rank(r.s, c)->hist[b];
        for (int c = 0; c < r.C; c++) cg::this_cluster().map_shared_rank(r.s, c)->tot[b] = n;
    }
    r.sync();
}

// Where the prefix of {comp >= tau0} ends whose metric (number of tokens, or mass) first reaches `target`:
// the comp of its last token. The histogram of the logits' bins is in s->hist (this CTA's share).
__device__ u64 pick_border(PickRow& r, bool by_mass, double target, u64 tau0) {
    PickShared* s = r.s;
    const int tid = threadIdx.x;
    int lo_bin = 0, hi_bin = kPickBins - 1, level = 0, shift = 0;
    u64 chi = ~0ull, clo = 0ull;
    double above = 0.0;  // metric of what lies above the members
    while (true) {
        pick_total(r);
        // bounds of the metric up to each bin; two bins per thread
        double lo[2], hi[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int b = 2 * tid + i;
            const double n = (double)s->tot[b];
            lo[i] = hi[i] = n;
            if (by_mass) {
                if (level == 0) {
                    const double step = kPickSpan / kPickBins;
                    hi[i] = n * exp2(-step * b) * kOne * (1.0 + 1e-4);
                    lo[i] = b == kPickBins - 1 ? 0.0 : n * exp2(-step * (b + 1)) * kOne * (1.0 - 1e-4);
                } else {
                    const u64 top = chi - ((u64)b << shift), span = ((u64)1 << shift) - 1ull;
                    hi[i] = n * (double)r.weight(pick_value(top));
                    lo[i] = n * (double)r.weight(pick_value(top > span ? top - span : 0ull));
                }
            }
        }
        double* red = reinterpret_cast<double*>(s->red);
        const double cl1 = pick_scan(lo[0] + lo[1], red) + above, cl0 = cl1 - lo[1];
        const double ch1 = pick_scan(hi[0] + hi[1], red) + above, ch0 = ch1 - hi[1];
        if (tid == 0) s->b1 = s->b2 = kPickBins - 1;
        __syncthreads();
        // sums of doubles may be off by a few parts in 2^53 per bin
        const double early = target * (1.0 - 1e-12), late = by_mass ? target * (1.0 + 1e-12) : target;
        if (ch1 >= early) atomicMin(&s->b1, ch0 >= early ? 2 * tid : 2 * tid + 1);
        if (cl1 >= late) atomicMin(&s->b2, cl0 >= late ? 2 * tid : 2 * tid + 1);
        if (tid == 0) s->count = 0u;
        __syncthreads();
        const int b1 = s->b1, b2 = max(s->b2, s->b1);
        u64 n = 0ull;
        for (int b = b1 + tid; b <= b2; b += kPickThreads) n += s->tot[b];
        n = pick_reduce(n, s->red, pick_add);
        const u64 chi1 = level == 0 ? ~0ull : chi - ((u64)b1 << shift);
        const u64 end = (u64)(b2 + 1) << shift;
        const u64 clo1 = level == 0 ? 0ull : chi - clo < end ? clo : chi - end + 1ull;
        if (level == 0) {
            lo_bin = b1;
            hi_bin = b2;
        }
        const bool fits = n <= (u64)kPickList;
        // what lies above the members, exactly; the members themselves, or their range
        u64 up = 0ull, first = ~0ull, last = 0ull;
        for (int i = r.w0; i < r.w1; i += 128) {
            float x[4];
            r.load(i + 4 * (tid & 31), x);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const u64 comp = pick_comp(x[j], i + 4 * (tid & 31) + j);
                bool in = x[j] > -INFINITY && comp >= tau0, over = false;
                if (in) {
                    const int b = r.bin(x[j]);
                    over = b < lo_bin || (b <= hi_bin && comp > chi1);
                    in = !over && b <= hi_bin && comp >= clo1;
                    if (over) up += by_mass ? r.weight(x[j]) : 1ull;
                    if (in) {
                        first = pick_min(first, comp);
                        last = pick_max(last, comp);
                    }
                }
                if (fits) pick_append(s, in, comp);
            }
        }
        above = (double)pick_sum(r, up);
        if (fits) {
            const int total = pick_collect(r);
            r.sync();
            if (r.rank == 0) {
                const int size = pick_pow2(max(total, 1));
                for (int i = total + tid; i < size; i += kPickThreads) s->list[i] = 0ull;
                pick_sort(s->list, size);
                // the first one at which the running metric reaches the target
                const int per = (size + kPickThreads - 1) / kPickThreads, i0 = min(total, tid * per);
                const int i1 = min(total, i0 + per);
                u64 sum = 0ull;
                for (int i = i0; i < i1; i++) sum += by_mass ? r.weight(pick_value(s->list[i])) : 1ull;
                const u64 incl = pick_scan(sum, s->red);
                u64 run = (u64)above + incl - sum;
                if (tid == 0) s->b1 = max(total - 1, 0);
                __syncthreads();
                if (i1 > i0 && (double)run < target && (double)(run + sum) >= target) {
                    int i = i0;
                    for (; i < i1 - 1; i++) {
                        run += by_mass ? r.weight(pick_value(s->list[i])) : 1ull;
                        if ((double)run >= target) break;
                    }
                    atomicMin(&s->b1, i);
                } else if (i1 > i0 && (double)run >= target) {
                    atomicMin(&s->b1, i0);  // reached before: the first token, at least
                }
                __syncthreads();
                if (tid == 0) {
                    const u64 tau = s->list[s->b1];
                    for (int c = 0; c < r.C; c++)
                        (r.C > 1 ? cg::this_cluster().map_shared_rank(s, c) : s)->tau = tau;
                }
            }
            r.sync();
            return s->tau;
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
        level++;
        shift = 0;
        while (((chi - clo) >> shift) >= (u64)kPickBins) shift++;
        for (int b = tid; b < kPickBins; b += kPickThreads) s->hist[b] = 0u;
        __syncthreads();
        for (int i = r.w0; i < r.w1; i += 128) {
            float x[4];
            r.load(i + 4 * (tid & 31), x);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const u64 comp = pick_comp(x[j], i + 4 * (tid & 31) + j);
                if (!(x[j] > -INFINITY) || comp < tau0 || comp < clo || comp > chi) continue;
                const int b = r.bin(x[j]);
                if (b >= lo_bin && b <= hi_bin) atomicAdd(&s->hist[(chi - comp) >> shift], 1u);
            }
        }
    }
}

__device__ __forceinline__ void pick_write(const PickArgs& a, int row, int id, float p) {
    a.ids[row] = id;
    if (a.probs) a.probs[row] = p;
}

// CTA 0 of the row: `n` tokens in s->list, the top-k among them: filters, draw.
__device__ void pick_short(const PickArgs& a, PickRow& r, int row, int n, int K, float P, double mp) {
    PickShared* s = r.s;
    const int tid = threadIdx.x;
    const int size = pick_pow2(n);
    for (int i = n + tid; i < size; i += kPickThreads) s->list[i] = 0ull;
    pick_sort(s->list, size);
    n = min(n, K);
    // two tokens per thread
    u64 w[2], c[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        c[i] = 2 * tid + i < n ? s->list[2 * tid + i] : 0ull;
        w[i] = 2 * tid + i < n ? r.weight(pick_value(c[i])) : 0ull;
    }
    u64 incl = pick_scan(w[0] + w[1], s->red);
    const u64 M = pick_reduce(incl, s->red, pick_max);
    const double need = P < 1.0f ? (double)P * (double)M : (double)~0ull;
    const u64 before[2] = {incl - w[0] - w[1], incl - w[1]};
    u64 kept = 0ull;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int at = 2 * tid + i;
        const bool keep = w[i] > 0ull && (at == 0 || (double)before[i] < need) && (double)w[i] >= mp * kOne;
        if (at < kPickTopK) s->w[at] = keep ? w[i] : 0ull;
        kept += keep;
    }
    const int m = (int)pick_reduce(kept, s->red, pick_add);  // they are the first m
    // in index order
    const int msize = pick_pow2(m);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int at = 2 * tid + i;
        if (at < msize) s->list[at] = at < m ? (c[i] << 32 | (u64)at) : 0ull;
    }
    pick_sort(s->list, msize);
    u64 ord[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        ord[i] = 2 * tid + i < m ? s->list[2 * tid + i] : 0ull;
        w[i] = 2 * tid + i < m ? s->w[(uint32_t)ord[i]] : 0ull;
    }
    incl = pick_scan(w[0] + w[1], s->red);
    const u64 S = pick_reduce(incl, s->red, pick_max);
    const double target = (double)a.u[row] * (double)S;
    u64 run = incl - w[0] - w[1];
    const bool inside = !((double)run > target) && ((double)incl > target || incl == S);
    if (w[0] > 0ull && (inside || (run == 0ull && (double)run > target))) {
        int i = 0;
        if (w[1] > 0ull && !((double)(run + w[0]) > target)) i = 1;
        pick_write(a, row, pick_index(ord[i] >> 32), (float)((double)w[i] / (double)S));
    }
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
    const double mp = a.min_p ? fmin((double)a.min_p[row], 1.0) : 0.0;
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
    const u64* x = r.exchange(top);
    for (int i = 0; i < C; i++) top = pick_max(top, x[i]);
    if (top == 0ull || !(Tf > 0.0f)) {
        if (r.rank == 0 && tid == 0) pick_write(a, row, top ? pick_index(top) : -1, top ? 1.0f : 0.0f);
        return;
    }
    r.mx = pick_value(top);
    r.c = 1.44269504088896340736 / (double)Tf;
    r.bin_scale = (float)(r.c * (kPickBins / (double)kPickSpan));

    if (K > 0 && K <= kPickTopK && K < V) {
        // the k-th largest of this CTA's maxima: at least k logits are as large
#pragma unroll
        for (int j = 0; j < 4; j++) s->list[4 * tid + j] = (u64)f32_order_key(m4[j] + 0.0f) << 32;
        pick_sort(s->list, 4 * kPickThreads);
        u64 bound = s->list[K - 1];
        const u64* b = r.exchange(bound);
        for (int i = 0; i < C; i++) bound = pick_max(bound, b[i]);
        for (int i = r.w0; i < r.w1; i += 128) {
            float q[4];
            r.load(i + 4 * lane, q);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const u64 comp = pick_comp(q[j], i + 4 * lane + j);
                pick_append(s, q[j] > -INFINITY && comp >= bound, comp);
            }
        }
        const int n = pick_collect(r);
        r.sync();
        if (n >= 0) {
            if (r.rank == 0) pick_short(a, r, row, n, K, P, mp);
            return;
        }
    }

    u64 tau = 0ull;
    const bool by_k = K > 0 && K < V, by_p = P < 1.0f;
    for (int pass = by_k ? 0 : 1; pass < (by_p ? 2 : 1); pass++) {
        // histogram of the logits' bins among {comp >= tau}, and their mass for top-p
        for (int b = tid; b < kPickBins; b += kPickThreads) s->hist[b] = 0u;
        __syncthreads();
        u64 mass = 0ull;
        for (int i = r.w0; i < r.w1; i += 128) {
            float q[4];
            r.load(i + 4 * lane, q);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (!(q[j] > -INFINITY) || pick_comp(q[j], i + 4 * lane + j) < tau) continue;
                atomicAdd(&s->hist[r.bin(q[j])], 1u);
                if (pass == 1) mass += r.weight(q[j]);
            }
        }
        double target = (double)K;
        if (pass == 1) target = (double)P * (double)pick_sum(r, mass);
        tau = pick_border(r, pass == 1, target, tau);
    }

    // sums of the kept weights by warp, in index order
    auto kept = [&](float q, int i) -> u64 {
        if (!(q > -INFINITY) || pick_comp(q, i) < tau) return 0ull;
        const u64 w = r.weight(q);
        return (double)w >= mp * kOne ? w : 0ull;
    };
    u64 sum = 0ull;
    for (int i = r.w0; i < r.w1; i += 128) {
        float q[4];
        r.load(i + 4 * lane, q);
#pragma unroll
        for (int j = 0; j < 4; j++) sum += kept(q[j], i + 4 * lane + j);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
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
    for (int i = r.w0; i < r.w1; i += 128) {
        float q[4];
        r.load(i + 4 * lane, q);
        u64 w[4], own = 0ull;
#pragma unroll
        for (int j = 0; j < 4; j++) own += w[j] = kept(q[j], i + 4 * lane + j);
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
            mine = i + 4 * lane + j;
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

// CTAs of a row: as many as fill the machine once at two CTAs per SM, while a
// CTA keeps 4096 logits or more.
int launch_pick(const PickArgs& a, cudaStream_t s) {
    if (a.rows == 0) return JYC_OK;
    const int sms = sm_count();
    if (sms == 0) return cuda_fail(cudaErrorNoDevice, "sample_batch: device query");
    int C = 1;
    while (C < kPickMaxCluster && (long long)a.rows * 2 * C <= 2 * sms && a.V / (2 * C) >= 4096) C *= 2;
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
