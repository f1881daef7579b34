// paged4.cu — K/V cache in pages at 4 bits a value: groups of 32 dims with an fp16 step and lowest value.
// Rows are quantised as they are written, read back as fp32, attended over by one new token per sequence
// (the scores and softmax of attention_q8, libs/model_libs/attention/attention_q8.h:38-184), which leaves
// each key's weight on it, and the rows of least weight are left behind.
#include "paged4.cuh"
#include "ptx.cuh"

#include <algorithm>
#include <climits>

namespace jyc {

namespace {

__device__ __forceinline__ void p4_flag(const PagedKV4& kv, int bit) {
    if ((*(volatile int*)kv.err & bit) == 0) atomicOr(kv.err, bit);
}
// Table entry of position `pos` >= 0 of sequence `seq`, -1 (and the error word) when the sequence or the position is
// out of range; *slot: its place there.
__device__ __forceinline__ int p4_entry(const PagedKV4& kv, int seq, int pos, int* slot) {
    const int idx = kv.by_page(pos);
    *slot = pos - idx * kv.p.page_size;
    if (seq < 0 || seq >= kv.num_seqs || idx >= kv.table_stride) {
        p4_flag(kv, kPagedErrPos);
        return -1;
    }
    const int page = __ldg(kv.table + (size_t)seq * kv.table_stride + idx);
    return page == -1 ? INT_MIN : page;  // -1: already flagged
}
// Whether an entry is a page; flags one that is not.
__device__ __forceinline__ bool p4_valid(const PagedKV4& kv, int page) {
    if (page >= 0 && page < kv.p.num_pages) return true;
    if (page != -1) p4_flag(kv, kPagedErrPage);
    return false;
}
__device__ __forceinline__ size_t p4_off(const jyc_kv_pages_q4& p, int page, int slot, int h) {
    return (size_t)((long long)page * p.page_stride + (long long)slot * p.pos_stride + (long long)h * p.head_stride);
}
__device__ __forceinline__ size_t p4_poff(const jyc_kv_pages_q4& p, int page, int slot, int h) {  // in pairs
    return (size_t)((long long)page * p.ppage_stride + (long long)slot * p.ppos_stride + (long long)h * p.phead_stride);
}
__device__ __forceinline__ size_t p4_moff(const jyc_kv_pages_q4& p, int page, int slot, int h) {
    return (size_t)((long long)page * p.mpage_stride + (long long)slot * p.mpos_stride + (long long)h * p.mhead_stride);
}

__device__ __forceinline__ float4 p4_load4(const float* p, bool vec) {
    if (vec) return __ldg(reinterpret_cast<const float4*>(p));
    return make_float4(__ldg(p), __ldg(p + 1), __ldg(p + 2), __ldg(p + 3));
}

// step and lowest value of a group whose values lie in lo .. hi, as (step, low) halves in one word
__device__ __forceinline__ uint32_t p4_params(float lo, float hi) {
    if (!(hi >= lo)) lo = hi = 0.0f;  // no number among them
    lo = fminf(fmaxf(lo, -65504.0f), 65504.0f);
    hi = fminf(fmaxf(hi, -65504.0f), 65504.0f);
    const __half low = __float2half_rn(lo), step = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.0f));
    return (uint32_t)__half_as_ushort(step) | (uint32_t)__half_as_ushort(low) << 16;
}
__device__ __forceinline__ float p4_step(uint32_t p) { return __half2float(__ushort_as_half((unsigned short)p)); }
__device__ __forceinline__ float p4_low(uint32_t p) { return __half2float(__ushort_as_half((unsigned short)(p >> 16))); }
__device__ __forceinline__ uint32_t p4_q(float x, float low, float inv) {
    return (uint32_t)min(max(__float2int_rn(__fmul_rn(__fsub_rn(x, low), inv)), 0), 15);
}

// ---------------------------------------------------------------------------
// Append and read back: a warp takes kP4Units * (32 / LANES) heads of K or of V
// of one row. LANES lanes hold a head, QUADS quads of dims each; a group of 32
// dims is 8 neighbouring lanes, so its range is three exchanges and its 16 bytes
// four words of the lower four lanes (whose high bits come from the upper four).
constexpr int kP4Units = 4, kP4Threads = 128;

struct P4Row {
    int row, head;  // first head of this lane
    bool is_k;
    int page, slot;  // page: as p4_entry returns it, -1: nothing to do
    int pos;
};
template <int LANES>
__device__ __forceinline__ P4Row p4_row(int rows, int chunks, const FastDiv& by_row, const int* row_seq,
                                        const int* row_pos, const PagedKV4& kv) {
    const int w = blockIdx.x * (kP4Threads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    P4Row x;
    x.row = by_row(w);
    const int r = w - x.row * 2 * chunks;
    x.is_k = r < chunks;
    x.head = (x.is_k ? r : r - chunks) * kP4Units * (32 / LANES) + lane / LANES;
    x.page = -1;
    x.slot = 0;
    x.pos = -1;
    if (x.row >= rows) return x;
    x.pos = __ldg(row_pos + x.row);
    const int seq = row_seq ? __ldg(row_seq + x.row) : x.row;
    if (x.pos >= 0) x.page = p4_entry(kv, seq, x.pos, &x.slot);
    return x;
}

template <int LANES, int QUADS>
__global__ void __launch_bounds__(kP4Threads) paged4_append_kernel(const float* K, const float* V, int ld, int rows,
                                                                   int KV, int hd, const int* row_seq,
                                                                   const int* row_pos, const int* rope_pos,
                                                                   PagedKV4 kv, RopeView rope, int chunks,
                                                                   FastDiv by_row, bool vec, bool wide_rope) {
    constexpr int SIDE = 32 / LANES;
    const int sub = threadIdx.x & (LANES - 1), nq = hd >> 2, groups = (hd + 31) >> 5;
    const P4Row x = p4_row<LANES>(rows, chunks, by_row, row_seq, row_pos, kv);
    if (x.page == -1) return;
    int turn = x.pos;
    if (rope.cos_t) {
        // a row that cannot turn is not written: neither its K nor its V
        if (rope_pos) turn = __ldg(rope_pos + x.row);
        if (turn < 0 || turn >= rope.len) {
            p4_flag(kv, kPagedErrRope);
            return;
        }
    }
    const bool rot = rope.cos_t && x.is_k;
    float4 v[kP4Units][QUADS];
    const float* src = (x.is_k ? K : V) + (size_t)x.row * ld + (size_t)x.head * hd;
#pragma unroll
    for (int i = 0; i < kP4Units; i++)
#pragma unroll
        for (int t = 0; t < QUADS; t++) {
            const int qd = sub + LANES * t;
            const float* head = src + i * SIDE * hd;
            if (qd >= nq || x.head + i * SIDE >= KV)
                v[i][t] = make_float4(0.f, 0.f, 0.f, 0.f);
            else if (rot)
                v[i][t] = turned4(head, 4 * qd, rope, turn, wide_rope);
            else
                v[i][t] = p4_load4(head + 4 * qd, vec);
        }
    if (!p4_valid(kv, x.page)) return;
    uint8_t* dst = (x.is_k ? kv.p.k : kv.p.v) + p4_off(kv.p, x.page, x.slot, x.head);
    uint32_t* par = reinterpret_cast<uint32_t*>(x.is_k ? kv.p.kp : kv.p.vp) + p4_poff(kv.p, x.page, x.slot, x.head);
#pragma unroll
    for (int i = 0; i < kP4Units; i++) {
        const bool live = x.head + i * SIDE < KV;
#pragma unroll
        for (int t = 0; t < QUADS; t++) {
            const int qd = sub + LANES * t, group = qd >> 3;
            const float4 a = v[i][t];
            float lo = INFINITY, hi = -INFINITY;
            if (qd < nq) {
                lo = fminf(fminf(fminf(fminf(lo, a.x), a.y), a.z), a.w);
                hi = fmaxf(fmaxf(fmaxf(fmaxf(hi, a.x), a.y), a.z), a.w);
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) {
                lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
                hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            }
            const uint32_t p = p4_params(lo, hi);
            const float step = p4_step(p), low = p4_low(p), inv = step > 0.0f ? __fdiv_rn(1.0f, step) : 0.0f;
            uint32_t w = 0u;
            if (qd < nq)
                w = p4_q(a.x, low, inv) | p4_q(a.y, low, inv) << 8 | p4_q(a.z, low, inv) << 16 | p4_q(a.w, low, inv) << 24;
            const uint32_t up = __shfl_xor_sync(0xffffffffu, w, 4);
            if (!live || group >= groups) continue;
            if ((sub & 7) < 4)
                *reinterpret_cast<uint32_t*>(dst + i * SIDE * kv.p.head_stride + 16 * group + 4 * (sub & 3)) = w | up << 4;
            if ((sub & 7) == 0) par[i * SIDE * kv.p.phead_stride + group] = p;
        }
        if (live && x.is_k && sub == 0 && kv.p.mass)
            kv.p.mass[p4_moff(kv.p, x.page, x.slot, x.head + i * SIDE)] = 0.0f;
    }
}

template <int LANES, int QUADS>
__global__ void __launch_bounds__(kP4Threads) paged4_read_kernel(float* K, float* V, int ld, int rows, int KV, int hd,
                                                                 const int* row_seq, const int* row_pos, PagedKV4 kv,
                                                                 int chunks, FastDiv by_row, bool vec) {
    constexpr int SIDE = 32 / LANES;
    const int sub = threadIdx.x & (LANES - 1), nq = hd >> 2;
    const P4Row x = p4_row<LANES>(rows, chunks, by_row, row_seq, row_pos, kv);
    if (x.page == -1 || !p4_valid(kv, x.page)) return;
    const uint8_t* src = (x.is_k ? kv.p.k : kv.p.v) + p4_off(kv.p, x.page, x.slot, x.head);
    const uint32_t* par =
        reinterpret_cast<const uint32_t*>(x.is_k ? kv.p.kp : kv.p.vp) + p4_poff(kv.p, x.page, x.slot, x.head);
    uint32_t w[kP4Units][QUADS], p[kP4Units][QUADS];
#pragma unroll
    for (int i = 0; i < kP4Units; i++)
#pragma unroll
        for (int t = 0; t < QUADS; t++) {
            const int qd = sub + LANES * t;
            const bool live = x.head + i * SIDE < KV && qd < nq;
            w[i][t] = live ? *reinterpret_cast<const uint32_t*>(src + i * SIDE * kv.p.head_stride + 16 * (qd >> 3) + 4 * (qd & 3))
                           : 0u;
            p[i][t] = live ? par[i * SIDE * kv.p.phead_stride + (qd >> 3)] : 0u;
        }
    float* dst = (x.is_k ? K : V) + (size_t)x.row * ld + (size_t)x.head * hd;
#pragma unroll
    for (int i = 0; i < kP4Units; i++) {
        if (x.head + i * SIDE >= KV) continue;
#pragma unroll
        for (int t = 0; t < QUADS; t++) {
            const int qd = sub + LANES * t;
            if (qd >= nq) continue;
            const uint32_t b = (qd & 4 ? w[i][t] >> 4 : w[i][t]) & 0x0F0F0F0Fu;
            const float step = p4_step(p[i][t]), low = p4_low(p[i][t]);
            float f[4];
            u8x4_to_f32(b ^ 0x80808080u, f);
#pragma unroll
            for (int j = 0; j < 4; j++) f[j] = __fmaf_rn(step, f[j], low);
            float* to = dst + i * SIDE * hd + 4 * qd;
            if (vec)
                *reinterpret_cast<float4*>(to) = make_float4(f[0], f[1], f[2], f[3]);
            else
#pragma unroll
                for (int j = 0; j < 4; j++) to[j] = f[j];
        }
    }
}

// ---------------------------------------------------------------------------
// Attention of one new token per sequence.
__device__ __forceinline__ int p4_len(const PagedAttn4& a, int b) {
    int len = a.lens[b];
    if (len <= 0) return 0;
    const int cap = a.kv.table_stride * a.kv.p.page_size;
    if (len > cap) {
        p4_flag(a.kv, kPagedErrPos);
        len = cap;
    }
    if (a.rope.cos_t) {
        const int pos = a.rope_pos ? a.rope_pos[b] : len - 1;
        if (pos < 0 || pos >= a.rope.len) {
            p4_flag(a.kv, kPagedErrRope);
            len = 0;
        }
    }
    return len;
}

constexpr int kP4MaxGroups = 8;
// A warp per key, a lane per dim of each group; a CTA per sequence and query head.
__device__ __forceinline__ float p4_simple_score(const PagedAttn4& a, const float* qv, int page, int slot, int kvh,
                                                 int lane) {
    const int groups = (a.hd + 31) / 32;
    const uint8_t* row = a.kv.p.k + p4_off(a.kv.p, page, slot, kvh);
    const uint32_t* par = reinterpret_cast<const uint32_t*>(a.kv.p.kp) + p4_poff(a.kv.p, page, slot, kvh);
    float s = 0.0f;
    for (int g = 0; g < groups; g++) {
        const int q = row[16 * g + (lane & 15)] >> (lane & 16 ? 4 : 0) & 15;
        s += qv[32 * g + lane] * __fmaf_rn(p4_step(par[g]), (float)q, p4_low(par[g]));
        // 0, or NaN where a parameter of K or V is not finite
        const uint32_t pv = reinterpret_cast<const uint32_t*>(a.kv.p.vp)[p4_poff(a.kv.p, page, slot, kvh) + g];
        const float all = p4_step(par[g]) * 0.0f + p4_low(par[g]) * 0.0f + p4_step(pv) * 0.0f + p4_low(pv) * 0.0f;
        s += all;
    }
    return warp_sum(s);
}
__device__ __forceinline__ float p4_simple_query(const PagedAttn4& a, int b, int h, int len, float* s_q) {
    const int lane = threadIdx.x & 31;
    __shared__ float s_scale;
    if (threadIdx.x < 32) {
        float x[kP4MaxGroups], amax = 0.0f;
        const float* q = a.Q + (size_t)b * a.ldq + (size_t)h * a.hd;
        const int pos = a.rope_pos ? a.rope_pos[b] : len - 1;
        for (int g = 0; g < kP4MaxGroups; g++) {
            const int d = 32 * g + lane;
            x[g] = 0.0f;
            if (d >= a.hd) continue;
            if (a.rope.cos_t) {
                const float4 y = turned4(q, d & ~3, a.rope, pos, false);
                x[g] = (d & 3) == 0 ? y.x : (d & 3) == 1 ? y.y : (d & 3) == 2 ? y.z : y.w;
            } else {
                x[g] = q[d];
            }
            amax = fmaxf(amax, fabsf(x[g]));
        }
        amax = warp_max(amax);
        for (int g = 0; g < kP4MaxGroups; g++) s_q[32 * g + lane] = (float)q8_round(x[g], q8_inv(amax));
        if (lane == 0) s_scale = __fmul_rn(q8_scale(amax), a.scale);
    }
    __syncthreads();
    return s_scale;
}
__global__ void __launch_bounds__(128) paged4_attention_simple(PagedAttn4 a, float2* stat) {
    __shared__ float s_q[32 * kP4MaxGroups], s_o[4][32 * kP4MaxGroups], s_m[4], s_l[4];
    const int b = blockIdx.x / a.H, h = blockIdx.x % a.H, kvh = h / (a.H / a.KV);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, groups = (a.hd + 31) / 32;
    const int len = p4_len(a, b);
    float* out = a.out + (size_t)b * a.ldo + (size_t)h * a.hd;
    if (len == 0) {
        for (int d = threadIdx.x; d < a.hd; d += 128) out[d] = 0.0f;
        return;
    }
    const float scale = p4_simple_query(a, b, h, len, s_q);
    float m = -INFINITY, l = 0.0f, o[kP4MaxGroups] = {};
    for (int j = warp; j < len; j += 4) {
        int slot;
        const int page = p4_entry(a.kv, b, j, &slot);
        if (!p4_valid(a.kv, page)) continue;
        const float s = __fmul_rn(p4_simple_score(a, s_q, page, slot, kvh, lane), scale);
        const float nm = m == m && s == s ? fmaxf(m, s) : NAN, f = m == -INFINITY ? 0.0f : __expf(m - nm), p = expf(s - nm);
        l = l * f + p;
        const uint8_t* row = a.kv.p.v + p4_off(a.kv.p, page, slot, kvh);
        const uint32_t* par = reinterpret_cast<const uint32_t*>(a.kv.p.vp) + p4_poff(a.kv.p, page, slot, kvh);
        for (int g = 0; g < groups; g++) {
            const int q = row[16 * g + (lane & 15)] >> (lane & 16 ? 4 : 0) & 15;
            o[g] = o[g] * f + p * __fmaf_rn(p4_step(par[g]), (float)q, p4_low(par[g]));
        }
        m = nm;
    }
    for (int g = 0; g < kP4MaxGroups; g++) s_o[warp][32 * g + lane] = o[g];
    if (lane == 0) {
        s_m[warp] = m;
        s_l[warp] = l;
    }
    __syncthreads();
    float M = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3])), L = 0.0f;
    for (int w = 0; w < 4; w++)
        if (s_m[w] != s_m[w]) M = NAN;
    for (int w = 0; w < 4; w++)
        if (!(s_m[w] == -INFINITY)) L += s_l[w] * expf(s_m[w] - M);
    for (int d = threadIdx.x; d < a.hd; d += 128) {
        float v = 0.0f;
        for (int w = 0; w < 4; w++)
            if (!(s_m[w] == -INFINITY)) v += s_o[w][d] * expf(s_m[w] - M);
        out[d] = L == 0.0f ? 0.0f : v / L;
    }
    if (stat && threadIdx.x == 0) stat[blockIdx.x] = make_float2(M, L);
}
__global__ void __launch_bounds__(128) paged4_mass_simple(PagedAttn4 a, const float2* stat, float* sums) {
    __shared__ float s_q[32 * kP4MaxGroups];
    const int b = blockIdx.x / a.KV, kvh = blockIdx.x % a.KV, group = a.H / a.KV;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int len = p4_len(a, b);
    if (len == 0) return;
    for (int i = 0; i < group; i++) {
        const int h = kvh * group + i;
        __syncthreads();
        const float scale = p4_simple_query(a, b, h, len, s_q);
        const float2 ml = stat[b * a.H + h];
        for (int j = warp; j < len; j += 4) {
            int slot;
            const int page = p4_entry(a.kv, b, j, &slot);
            if (!p4_valid(a.kv, page)) continue;
            const float s = __fmul_rn(p4_simple_score(a, s_q, page, slot, kvh, lane), scale);
            if (lane == 0) {
                float* sum = sums + (size_t)blockIdx.x * a.kv.table_stride * a.kv.p.page_size + j;
                const float w = (i == 0 ? 0.0f : *sum) + expf(s - ml.x) / ml.y;
                if (i < group - 1)
                    *sum = w;
                else
                    atomicAdd(a.kv.p.mass + p4_moff(a.kv.p, page, slot, kvh), w);
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Eviction: a CTA finds which rows a kv head of a sequence keeps, then warps
// copy them.
constexpr int kEvThreads = 1024;

// larger mass -> larger key; NaN below every number, -0 as 0
__device__ __forceinline__ uint32_t ev_key(float m) { return f32_order_key(m + 0.0f); }

__global__ void __launch_bounds__(kEvThreads) paged4_select_kernel(PagedEvict4 e) {
    __shared__ int s_hist[256], s_digit, s_above, s_scan[kEvThreads / 32][2];
    const int b = blockIdx.x / e.KV, h = blockIdx.x % e.KV, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int len = max(e.lens[b], 0);
    const int cap = e.kv.table_stride * e.kv.p.page_size;
    if (len > cap) {
        p4_flag(e.kv, kPagedErrPos);
        len = cap;
    }
    int* kept = e.kept + (size_t)blockIdx.x * e.budget;
    const int n = min(len, e.budget);
    if (h == 0 && tid == 0) e.new_lens[b] = n;
    if (len <= e.budget) {
        for (int i = tid; i < e.budget; i += kEvThreads) kept[i] = i < len ? i : -1;
        return;
    }
    const int old = len - e.recent, want = e.budget - e.recent;  // want < old
    auto key = [&](int i) {
        int slot;
        const int page = p4_entry(e.kv, b, i, &slot);
        return p4_valid(e.kv, page) ? ev_key(e.kv.p.mass[p4_moff(e.kv.p, page, slot, h)]) : 0u;
    };
    uint32_t prefix = 0u;
    int left = want;  // of those that share the prefix, how many are kept
    if (want > 0)
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += kEvThreads) s_hist[i] = 0;
            __syncthreads();
            for (int i = tid; i < old; i += kEvThreads) {
                const uint32_t k = key(i);
                if (shift == 24 || k >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&s_hist[k >> shift & 255], 1);
            }
            __syncthreads();
            if (tid == 0) {
                int above = 0, d = 255;
                while (above + s_hist[d] < left) above += s_hist[d--];
                s_digit = d;
                s_above = above;
            }
            __syncthreads();
            prefix |= (uint32_t)s_digit << shift;
            left -= s_above;
            __syncthreads();
        }
    // positions in order: those above the border, and the first `left` that equal it
    int base = 0, ties = 0;
    for (int i0 = 0; i0 < len; i0 += kEvThreads) {
        const int i = i0 + tid;
        const uint32_t k = want > 0 && i < old ? key(i) : 0u;
        const bool tie = want > 0 && i < old && k == prefix, sure = i < len && (i >= old || (want > 0 && k > prefix));
        const unsigned ties_w = __ballot_sync(0xffffffffu, tie);
        if (lane == 0) s_scan[warp][0] = __popc(ties_w);
        __syncthreads();
        int before = ties + __popc(ties_w & ((1u << lane) - 1u));
        for (int w = 0; w < kEvThreads / 32; w++) {
            if (w < warp) before += s_scan[w][0];
            ties += s_scan[w][0];
        }
        const bool keep = sure || (tie && before < left);
        const unsigned keep_w = __ballot_sync(0xffffffffu, keep);
        if (lane == 0) s_scan[warp][1] = __popc(keep_w);
        __syncthreads();
        int at = base + __popc(keep_w & ((1u << lane) - 1u));
        for (int w = 0; w < kEvThreads / 32; w++) {
            if (w < warp) at += s_scan[w][1];
            base += s_scan[w][1];
        }
        if (keep) kept[at] = i;
        __syncthreads();
    }
}

__global__ void __launch_bounds__(256) paged4_move_kernel(PagedEvict4 e) {
    const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (w >= (long long)e.kv.num_seqs * e.KV * e.budget) return;
    const int item = (int)(w / e.budget), to = (int)(w - (long long)item * e.budget), b = item / e.KV, h = item % e.KV;
    const int from = e.kept[w];
    if (from < 0) return;
    int ss, ds;
    const int sp = p4_entry(e.kv, b, from, &ss);
    PagedKV4 dst = e.kv;
    dst.table = e.new_table;
    dst.table_stride = e.new_stride;
    const int dp = p4_entry(dst, b, to, &ds);
    const bool ok = p4_valid(e.kv, sp) && p4_valid(e.kv, dp);
    if (!ok) return;
    const jyc_kv_pages_q4& p = e.kv.p;
    const size_t so = p4_off(p, sp, ss, h), to_ = p4_off(p, dp, ds, h);
    const size_t sq = p4_poff(p, sp, ss, h), dq = p4_poff(p, dp, ds, h);
    const int groups = (e.hd + 31) / 32;
    if (lane < 4 * groups) {
        reinterpret_cast<uint32_t*>(p.k + to_)[lane] = reinterpret_cast<const uint32_t*>(p.k + so)[lane];
        reinterpret_cast<uint32_t*>(p.v + to_)[lane] = reinterpret_cast<const uint32_t*>(p.v + so)[lane];
    }
    if (lane < groups) {
        reinterpret_cast<uint32_t*>(p.kp)[dq + lane] = reinterpret_cast<const uint32_t*>(p.kp)[sq + lane];
        reinterpret_cast<uint32_t*>(p.vp)[dq + lane] = reinterpret_cast<const uint32_t*>(p.vp)[sq + lane];
    }
    if (lane == 0) p.mass[p4_moff(p, dp, ds, h)] = p.mass[p4_moff(p, sp, ss, h)];
}

bool aligned16(const void* p, int ld) { return ((uintptr_t)p & 15) == 0 && (ld & 3) == 0; }

// The cache of rows r0, r0 + 1, ... when a row is its own sequence.
PagedKV4 shifted(PagedKV4 kv, const int* row_seq, int r0) {
    if (!row_seq) {
        kv.table += (size_t)r0 * kv.table_stride;
        kv.num_seqs -= r0;
    }
    return kv;
}

// Rows in launches of fewer than 2^30 warps. f(first row, rows, CTAs, warps that share K or V of a row).
template <class F>
int row_launches(int rows, int KV, int hd, F f) {
    const int lanes = hd <= 32 ? 8 : hd <= 64 ? 16 : 32, per = kP4Units * (32 / lanes), chunks = (KV + per - 1) / per;
    const int most = std::max(1, (1 << 30) / (2 * chunks)), warps = kP4Threads / 32;
    for (int r0 = 0; r0 < rows; r0 += most) {
        const int n = std::min(most, rows - r0);
        f(r0, n, (unsigned)(((long long)n * 2 * chunks + warps - 1) / warps), chunks);
        JYC_LAUNCHED();
        if (rows - r0 <= most) break;
    }
    return JYC_OK;
}

}  // namespace

int launch_paged4_append(const float* K, const float* V, int ld, int rows, int KV, int hd, const int* row_seq,
                         const int* row_pos, const int* rope_pos, const PagedKV4& kv, const RopeView& rope,
                         cudaStream_t s) {
    const bool vec = aligned16(K, ld) && aligned16(V, ld), wide = vec && rope_wide(rope);
    const auto kernel = hd <= 32    ? paged4_append_kernel<8, 1>
                        : hd <= 64  ? paged4_append_kernel<16, 1>
                        : hd <= 128 ? paged4_append_kernel<32, 1>
                                    : paged4_append_kernel<32, 2>;
    return row_launches(rows, KV, hd, [&](int r0, int n, unsigned grid, int chunks) {
        kernel<<<grid, kP4Threads, 0, s>>>(K + (size_t)r0 * ld, V + (size_t)r0 * ld, ld, n, KV, hd,
                                           row_seq ? row_seq + r0 : nullptr, row_pos + r0,
                                           rope_pos ? rope_pos + r0 : nullptr, shifted(kv, row_seq, r0), rope, chunks,
                                           fast_div(2 * chunks), vec, wide);
    });
}

int launch_paged4_read(float* K, float* V, int ld, int rows, int KV, int hd, const int* row_seq, const int* row_pos,
                       const PagedKV4& kv, cudaStream_t s) {
    const bool vec = aligned16(K, ld) && aligned16(V, ld);
    const auto kernel = hd <= 32    ? paged4_read_kernel<8, 1>
                        : hd <= 64  ? paged4_read_kernel<16, 1>
                        : hd <= 128 ? paged4_read_kernel<32, 1>
                                    : paged4_read_kernel<32, 2>;
    return row_launches(rows, KV, hd, [&](int r0, int n, unsigned grid, int chunks) {
        kernel<<<grid, kP4Threads, 0, s>>>(K + (size_t)r0 * ld, V + (size_t)r0 * ld, ld, n, KV, hd,
                                           row_seq ? row_seq + r0 : nullptr, row_pos + r0, shifted(kv, row_seq, r0),
                                           chunks, fast_div(2 * chunks), vec);
    });
}

size_t paged4_attention_workspace(int seqs, int H, int KV, int, int capacity) {
    return sm_count() ? 16 + sizeof(float2) * seqs * H + sizeof(float) * (size_t)seqs * KV * capacity : 0;
}

int launch_paged4_attention(const PagedAttn4& a, void* work, cudaStream_t s) {
    float2* stat = a.kv.p.mass ? static_cast<float2*>(work) : nullptr;
    paged4_attention_simple<<<a.kv.num_seqs * a.H, 128, 0, s>>>(a, stat);
    JYC_LAUNCHED();
    if (stat) {
        paged4_mass_simple<<<a.kv.num_seqs * a.KV, 128, 0, s>>>(
            a, stat, reinterpret_cast<float*>(stat + (size_t)a.kv.num_seqs * a.H));
        JYC_LAUNCHED();
    }
    return JYC_OK;
}

int launch_paged4_evict(const PagedEvict4& e, cudaStream_t s) {
    paged4_select_kernel<<<e.kv.num_seqs * e.KV, kEvThreads, 0, s>>>(e);
    JYC_LAUNCHED();
    const long long warps = (long long)e.kv.num_seqs * e.KV * e.budget;
    paged4_move_kernel<<<(unsigned)((warps + 7) / 8), 256, 0, s>>>(e);
    JYC_LAUNCHED();
    return JYC_OK;
}

}  // namespace jyc
