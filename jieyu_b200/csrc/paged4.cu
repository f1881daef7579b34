// paged4.cu — K/V cache in pages at 4 bits a value: groups of 32 dims with an fp16 step and lowest value.
// Rows are quantised as they are written, read back as fp32, attended over by one new token per sequence
// (the scores and softmax of attention_q8, libs/model_libs/attention/attention_q8.h:38-184), which leaves
// each key's weight on it, and the rows of least weight are left behind.
#include "paged4.cuh"
#include "follow.cuh"
#include "paged_line.cuh"
#include "ptx.cuh"
#include "tmap.cuh"

#include <algorithm>
#include <climits>
#include <numeric>

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
// ---------------------------------------------------------------------------
// Append and read back: a warp takes UNITS * (32 / LANES) heads of K or of V of one
// row, the loads of all units in flight. The bookkeeping of a row is shared.
constexpr int kP4Threads = 128;

struct P4Row {
    int row, head;  // first head of this lane
    bool is_k;
    int page, slot;  // page: as p4_entry returns it, -1: nothing to do
    int pos;
};
template <int LANES, int UNITS>
__device__ __forceinline__ P4Row p4_row(int rows, int chunks, const FastDiv& by_row, const int* row_seq,
                                        const int* row_pos, const PagedKV4& kv) {
    const int w = blockIdx.x * (kP4Threads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    P4Row x;
    x.row = by_row(w);
    const int r = w - x.row * 2 * chunks;
    x.is_k = r < chunks;
    x.head = (x.is_k ? r : r - chunks) * UNITS * (32 / LANES) + lane / LANES;
    x.page = -1;
    x.slot = 0;
    x.pos = -1;
    if (x.row >= rows) return x;
    x.pos = __ldg(row_pos + x.row);
    const int seq = row_seq ? __ldg(row_seq + x.row) : x.row;
    if (x.pos >= 0) x.page = p4_entry(kv, seq, x.pos, &x.slot);
    return x;
}

// four values as bytes 0 .. 15: held in range (a NaN as 0), then rounded by the sum with 1.5 * 2^23
__device__ __forceinline__ uint32_t p4_bytes(float4 x, float low, float inv) {
    auto q = [&](float v) {
        return __float_as_uint(__fadd_rn(fminf(fmaxf(__fmul_rn(__fsub_rn(v, low), inv), 0.0f), 15.0f), 12582912.0f));
    };
    return __byte_perm(__byte_perm(q(x.x), q(x.y), 0x0040), __byte_perm(q(x.z), q(x.w), 0x0040), 0x5410);
}

// Four lanes hold a group: lane i its dims 4 i .. 4 i + 3 and 16 more, whose numbers are the low and the high bits of its
// word; the group's range is two exchanges. Of four heads in flight each lane makes one's parameters and passes them on.
// Pairs that lie on quads turn by table entries that a lane reads once for all of its heads; others, which are rare, value
// by value (P4_ODD: 78 us behind a flushed L2 where quads take 40 to 48). Bound by its instructions, 84 a head of 128 and
// warp: 16384 rows of 8 x 128 33 us (floor 24), 45 where every lane makes the parameters of all heads, 60 with the
// rotation's form chosen value by value too, 72 with four dims a lane.
enum { P4_PLAIN = 0, P4_PAIRS = 1, P4_HALVES = 2, P4_ODD = 3 };  // how K turns
template <int LANES, int UNITS, int MODE>
__global__ void __launch_bounds__(kP4Threads) paged4_append_kernel(const float* K, const float* V, int ld, int rows,
                                                                   int KV, int hd, const int* row_seq,
                                                                   const int* row_pos, const int* rope_pos,
                                                                   PagedKV4 kv, RopeView rope, int chunks,
                                                                   FastDiv by_row, bool vec) {
    griddep_wait();
    constexpr int SIDE = 32 / LANES;
    const int sub = threadIdx.x & (LANES - 1), group = sub >> 2, d0 = 32 * group + 4 * (sub & 3), groups = (hd + 31) >> 5;
    const P4Row x = p4_row<LANES, UNITS>(rows, chunks, by_row, row_seq, row_pos, kv);
    if (x.page == -1) return;
    int turn = x.pos;
    if (MODE != P4_PLAIN) {
        // a row that cannot turn is not written: neither its K nor its V
        if (rope_pos) turn = __ldg(rope_pos + x.row);
        if (turn < 0 || turn >= rope.len) {
            p4_flag(kv, kPagedErrRope);
            return;
        }
    }
    const bool in0 = d0 < hd, in1 = d0 + 16 < hd;
    float4 v[UNITS][2];
    const float* src = (x.is_k ? K : V) + (size_t)x.row * ld + (size_t)x.head * hd;
#pragma unroll
    for (int i = 0; i < UNITS; i++)
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const bool in = (t ? in1 : in0) && x.head + i * SIDE < KV;
            const float* at = src + i * SIDE * hd + d0 + 16 * t;
            v[i][t] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (!in) continue;
            if (MODE == P4_ODD && x.is_k)
                v[i][t] = turned4(src + i * SIDE * hd, d0 + 16 * t, rope, turn, false);
            else
                v[i][t] = p4_load4(at, MODE == P4_PAIRS || MODE == P4_HALVES || vec);
        }
    if (MODE == P4_PAIRS && x.is_k) {
        float2 c[2], sn[2];
        const size_t tab = (size_t)turn * rope.half;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int d = d0 + 16 * t;
            const bool use = d < 2 * rope.half;
            c[t] = use ? __ldg(reinterpret_cast<const float2*>(rope.cos_t + tab + d / 2)) : make_float2(1.0f, 1.0f);
            sn[t] = use ? __ldg(reinterpret_cast<const float2*>(rope.sin_t + tab + d / 2)) : make_float2(0.0f, 0.0f);
        }
#pragma unroll
        for (int t = 0; t < 2; t++)
            if (d0 + 16 * t < 2 * rope.half)
#pragma unroll
                for (int i = 0; i < UNITS; i++) {
                    const float4 a = v[i][t];
                    turn_pair(a.x, a.y, c[t].x, sn[t].x, v[i][t].x, v[i][t].y);
                    turn_pair(a.z, a.w, c[t].y, sn[t].y, v[i][t].z, v[i][t].w);
                }
    }
    if (MODE == P4_HALVES && x.is_k) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int d = d0 + 16 * t;
            if (d >= 2 * rope.half) continue;
            const bool first = d < rope.half;
            const int other = first ? rope.half : -rope.half;
            const size_t tab = (size_t)turn * rope.half + (first ? d : d - rope.half);
            const float4 c = __ldg(reinterpret_cast<const float4*>(rope.cos_t + tab));
            const float4 sn = __ldg(reinterpret_cast<const float4*>(rope.sin_t + tab));
            float4 w[UNITS];
#pragma unroll
            for (int i = 0; i < UNITS; i++)
                w[i] = x.head + i * SIDE < KV ? p4_load4(src + i * SIDE * hd + d + other, true) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < UNITS; i++) {
                const float4 a = first ? v[i][t] : w[i], b = first ? w[i] : v[i][t];
                float4 r0, r1;
                turn_pair(a.x, b.x, c.x, sn.x, r0.x, r1.x);
                turn_pair(a.y, b.y, c.y, sn.y, r0.y, r1.y);
                turn_pair(a.z, b.z, c.z, sn.z, r0.z, r1.z);
                turn_pair(a.w, b.w, c.w, sn.w, r0.w, r1.w);
                v[i][t] = first ? r0 : r1;
            }
        }
    }
    if (!p4_valid(kv, x.page)) return;
    uint8_t* dst = (x.is_k ? kv.p.k : kv.p.v) + p4_off(kv.p, x.page, x.slot, x.head) + 4 * sub;
    uint32_t* par = reinterpret_cast<uint32_t*>(x.is_k ? kv.p.kp : kv.p.vp) + p4_poff(kv.p, x.page, x.slot, x.head) + group;
    float lo[UNITS], hi[UNITS], inv[UNITS];
    uint32_t p[UNITS];
#pragma unroll
    for (int i = 0; i < UNITS; i++) {
        const float4 a = v[i][0], c = v[i][1];
        lo[i] = INFINITY;
        hi[i] = -INFINITY;
        if (in0) {
            lo[i] = fminf(fminf(a.x, a.y), fminf(a.z, a.w));
            hi[i] = fmaxf(fmaxf(a.x, a.y), fmaxf(a.z, a.w));
        }
        if (in1) {
            lo[i] = fminf(lo[i], fminf(fminf(c.x, c.y), fminf(c.z, c.w)));
            hi[i] = fmaxf(hi[i], fmaxf(fmaxf(c.x, c.y), fmaxf(c.z, c.w)));
        }
    }
    // the group's range over its four lanes, then its parameters: of four units each lane makes (and stores) one's
    const int own = UNITS == 4 ? sub & 3 : 0;
    float low, high;
    if constexpr (UNITS == 4) {
        const bool b1 = sub & 2, b0 = sub & 1;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            lo[i] = fminf(b1 ? lo[i + 2] : lo[i], __shfl_xor_sync(0xffffffffu, b1 ? lo[i] : lo[i + 2], 2));
            hi[i] = fmaxf(b1 ? hi[i + 2] : hi[i], __shfl_xor_sync(0xffffffffu, b1 ? hi[i] : hi[i + 2], 2));
        }
        low = fminf(b0 ? lo[1] : lo[0], __shfl_xor_sync(0xffffffffu, b0 ? lo[0] : lo[1], 1));
        high = fmaxf(b0 ? hi[1] : hi[0], __shfl_xor_sync(0xffffffffu, b0 ? hi[0] : hi[1], 1));
    } else {
        static_assert(UNITS == 1 || UNITS == 4, "");
        low = fminf(lo[0], __shfl_xor_sync(0xffffffffu, lo[0], 1));
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, 2));
        high = fmaxf(hi[0], __shfl_xor_sync(0xffffffffu, hi[0], 1));
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 2));
    }
    p[0] = p4_params(low, high);
    inv[0] = p4_step(p[0]) > 0.0f ? __frcp_rn(p4_step(p[0])) : 0.0f;
    const int head = x.head + own * SIDE;
    if (head < KV && group < groups && (UNITS == 4 || (sub & 3) == 0)) {
        par[own * SIDE * kv.p.phead_stride] = p[0];
        if (x.is_k && sub < 4 && kv.p.mass) kv.p.mass[p4_moff(kv.p, x.page, x.slot, head)] = 0.0f;
    }
    if constexpr (UNITS == 4) {
        const uint32_t mine = p[0];
        const float inverse = inv[0];
#pragma unroll
        for (int i = 0; i < UNITS; i++) {
            p[i] = __shfl_sync(0xffffffffu, mine, i, 4);
            inv[i] = __shfl_sync(0xffffffffu, inverse, i, 4);
        }
    }
#pragma unroll
    for (int i = 0; i < UNITS; i++) {
        const float base = p4_low(p[i]);
        const uint32_t w = (in0 ? p4_bytes(v[i][0], base, inv[i]) : 0u) | (in1 ? p4_bytes(v[i][1], base, inv[i]) << 4 : 0u);
        if (x.head + i * SIDE < KV && group < groups) *reinterpret_cast<uint32_t*>(dst + i * SIDE * kv.p.head_stride) = w;
    }
}

// Eight neighbouring lanes read a group, two of them each word.
constexpr int kP4Units = 4;
template <int LANES, int QUADS>
__global__ void __launch_bounds__(kP4Threads) paged4_read_kernel(float* K, float* V, int ld, int rows, int KV, int hd,
                                                                 const int* row_seq, const int* row_pos, PagedKV4 kv,
                                                                 int chunks, FastDiv by_row, bool vec) {
    griddep_wait();
    constexpr int SIDE = 32 / LANES;
    const int sub = threadIdx.x & (LANES - 1), nq = hd >> 2;
    const P4Row x = p4_row<LANES, kP4Units>(rows, chunks, by_row, row_seq, row_pos, kv);
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
//
// Row j of a kv head is low_jg + step_jg q (group g of 32 dims). With the query as whole numbers x and their sums X_g:
// s_j = qs sum_g (step_jg (x . q)_jg + low_jg X_g) / sqrt(hd), out = sum_j p_j (low_jg + step_jg q) / sum_j p_j.
// Each product takes the form whose operands are exact on the tensor cores. Scores: keys are the rows, the query heads of a
// kv head the columns; the dots x . q of a group are one mma.m16n8k32 of bytes (nibbles masked out of the stored words), made
// floats by an exact subtraction and added with their step; low X is one mma.m16n8k16 of the stored (step, low) halves
// against (0, X), X as two halves. Values: rows are dims, the stored words turned by ldmatrix.trans, each nibble masked into
// a half (q - 8, or 16 times that) in two operations; the weight p_j step_jg as halves hi + lo, made from p's
// halves by three fp16 operations (the product rounded, what that left, the low half's share); p (low + 8 step) is one product of the
// stored halves. Each unit's product starts from zero and is added in fp32 with round to nearest (the tensor cores' own
// sums may truncate).
//
// A key counts by its weight, so that one that is large and hardly seen must not cost the others their bits. Steps are
// taken in units of 2^e of their group, which follow the units of keys up and down, so that a weight times a step stays
// within fp16; the weights of a unit whose keys all score low are taken 2^d up and its sums 2^d down again, so that its
// largest weight is 2^9 at least (2^5 of values within 2^4 of one another). Where the values of each group lie within 2^8 of
// one another (p4_fits) their steps are exact (or next to far larger lows), and fp16's roundings, 2^-19.7 a key at most, are
// small against sum p (|low| + 15 step), which is 2^4.9 at least (64 that all fall the same way: 2^-18). A unit whose keys
// lie further apart is added key by key in fp32. 131072 keys of 8 x 128: 60.4 us (59.0 with one e for all keys so far, where
// one step of 8736 made steps of 1e-4 zeros whatever its weight); behind a flushed L2 67, 81 with one key in 1000 far above
// the others, 210 with steps of 1e-4 to 0.1 in every unit.
//
// A step reads sum(len) * KV * 40 G bytes (G groups). The line of units, runs and joins are paged_line.cuh's; teams of
// warps take the same keys of neighbouring kv heads, whose rows lie side by side in [page][slot][kv head] (262144 keys of 8 x
// 128, without products: 95 us, 142 with every head at its own keys). Rows of 32 or 64 bytes come by tensor copies, others and
// all parameters by cp.async. The reference follows the maximum of the scores; the accumulators are rescaled only where it
// or a group's e moves.
//
// Measured: 131072 keys of 8 x 128 60 us (floor 26), 48 sequences of up to 8192 keys with their weights 98-111 us (floor
// 37), 513 keys of 2 x 64 14 us. At 131072 keys about 20 us pass before the first and behind the last key (launches, run
// search, page table, first copies; parts and the join); between them issue slots are 55 % busy, the warps waiting for one
// another's results in chains of products and exchanges (the copies without products take 45 us behind a flushed L2).
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

// Sizes of one instantiation: GP groups (the head size rounded up), HEADS query heads of a unit, rows by tensor copies.
template <int GP, int HEADS, bool TMA>
struct P4Cfg {
    using Args = PagedAttn4;
    static __device__ __forceinline__ int len(const PagedAttn4& a, int b) { return p4_len(a, b); }
    static constexpr bool STAT = true, TEAM = true;
    static constexpr bool WIDE = GP == 4 && HEADS > 8;
    static constexpr int U = GP <= 2 || WIDE ? 2 : 1;  // keys of a lane
    static constexpr int HDP = 32 * GP, TK = 32 * U;   // keys of a unit
    // few warps of long units against more of short ones: 131072 keys of 8 x 128, 4 heads each, 61.5 us with 12 warps of 32
    // keys, 62 with 8 of 64 (48 sequences of up to 8192 keys 96-103 and 102-104); with V as subnormal halves, which was 4 us
    // faster, 57, 58 and 70 with 16 of 32; 16 heads each, 65536 keys, 65 us with 8 of 64, 74 with 12 of 32; 64 sequences of
    // 2112 keys of 8 x 64, 4 heads each, 50 us with 12 warps of 64, 55 with 8. With 16 heads each the 168 registers of 12
    // warps do not hold a unit: behind a flushed L2 108 us, 98 with 8; 4 kv heads in pages of 5 80 and 63. (Heads above
    // 128 with 16 heads each spill 260 to 500 bytes a thread at 255 registers: 30000 keys of 4 x 256 take 76 us.)
    static constexpr int WARPS = GP <= 4 && HEADS <= 8 ? 12 : 8;
    static constexpr int ST = GP == 6 ? 3 : 2;
    static constexpr int E = HEADS <= 8 ? 1 : 2;  // n8 tiles of heads
    static constexpr int ROWS = HEADS;
    // rows of K and V: tensor copies swizzle their 16-byte chunks, else an odd number of chunks, so that the 8 rows of an
    // ldmatrix tile lie in distinct banks
    static constexpr int PITCH = 16 * GP + (TMA ? 0 : 16);
    static constexpr int PW = GP <= 4 ? 4 : 8;  // words of a key's parameters: whole 16 bytes
    static constexpr int VOFF = TK * PITCH, KPOFF = 2 * TK * PITCH, VPOFF = KPOFF + 4 * PW * TK;
    static constexpr int STAGE = VPOFF + 4 * PW * TK;
    static constexpr int PART = ROWS * (HDP + 2);  // floats of a partial: o, then (ref, l) per row
    static constexpr int SOFF = ST * STAGE;        // V's steps of the current unit
    static constexpr int RING = TMA ? (SOFF + 64 * GP * U + 1023) / 1024 * 1024 : SOFF + 64 * GP * U;
    static constexpr int SMEM = WARPS * RING + (TMA ? 1024 : 0);
    static_assert(PART * 4 <= RING, "a partial fits the ring");
    static_assert(!TMA || GP == 2 || GP == 4, "rows of 32 or 64 bytes");
    // byte of 16-byte chunk c of row r
    static __device__ __forceinline__ int at(int r, int c) {
        return r * PITCH + 16 * (!TMA ? c : GP == 4 ? c ^ ((r >> 1) & 3) : c ^ ((r >> 2) & 1));
    }
};
struct P4Maps {
    CUtensorMap k, v;
};
// Where the scores (base 2) of unit `t` of row of units `r` of a sequence lie, for the kernel that gathers the weights:
// [key][ROWS].
struct P4Scores {
    float* s;  // nullptr: no weights are gathered
    long long keys;  // floats of a row of units
};
__device__ __forceinline__ size_t p4_score_at(const P4Scores& sc, const PaPlan& pl, int b, int r, int t, int unit) {
    return (size_t)((long long)b * pl.units_row * pl.team + r) * sc.keys + (size_t)t * unit;
}
// two fp32 operations in one instruction
__device__ __forceinline__ void p4_add2(float& x, float& y, float a, float b) {
    asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tadd.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(a), "f"(b));
}
__device__ __forceinline__ void p4_mul2(float& x, float& y, float a, float b) {
    asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmul.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(a), "f"(b));
}
__device__ __forceinline__ void p4_fma2(float& x, float& y, float a, float b, float c, float d) {  // += (a, b) * (c, d)
    asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmov.b64 r, {%4, %5};\n\t"
        "fma.rn.f32x2 p, q, r, p;\n\tmov.b64 {%0, %1}, p;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(a), "f"(b), "f"(c), "f"(d));
}
__device__ __forceinline__ __half2 p4_h2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
__device__ __forceinline__ uint32_t p4_u(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }
// 2^k as a half (-24 <= k <= 15) and as a float
__device__ __forceinline__ uint32_t p4_half_pow2(int k) { return k >= -14 ? (uint32_t)(k + 15) << 10 : 1u << (k + 24); }
__device__ __forceinline__ float p4_pow2(int k) { return __uint_as_float((uint32_t)(127 + k) << 23); }
// What takes V's (step, low) of a group to units of 2^(e - 15), lows by eighths: both below 2 where they fit.
__device__ __forceinline__ uint32_t p4_units(int e) { return p4_half_pow2(15 - e) | p4_half_pow2(12 - e) << 16; }
// Whether a key's step and low keep all of their bits in units of 2^(e - 15): the step below 2 of them, low below 16, and
// the step at 2^-8 at least or low at 1.
__device__ __forceinline__ bool p4_fits(uint32_t par, int e) {
    const float step = fabsf(p4_step(par)), low = fabsf(p4_low(par));
    return step < p4_pow2(e - 14) && low < p4_pow2(e - 11) && (step >= p4_pow2(e - 23) || low >= p4_pow2(e - 15));
}
// the low (HIGH: the next 4) bits of each half as halves q - 8 (16 (q - 8)): 0x6400 | n is 1024 + n. (Left as they are, q 2^-24,
// they are exact too, but the tensor cores do not shift subnormals up before they align products: 10 of the sums' 24 bits
// went. Numbers around 0 keep the sums, which may be truncated, small.)
template <bool HIGH>
__device__ __forceinline__ uint32_t p4_whole(uint32_t x) {
    return p4_u(__hsub2(p4_h2((x & (HIGH ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u),
                        __half2half2(__ushort_as_half(HIGH ? 0x6480 : 0x6408))));
}
template <int N>
__device__ __forceinline__ void p4_words(const uint32_t* p, uint32_t (&w)[N]) {  // N even
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint4 x = *reinterpret_cast<const uint4*>(p + 4 * i);
            w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            const uint2 x = *reinterpret_cast<const uint2*>(p + 2 * i);
            w[2 * i] = x.x; w[2 * i + 1] = x.y;
        }
    }
}
// Parameters of neighbouring heads may share a sector, which other SMs want too: no hint.
template <int N>
__device__ __forceinline__ void p4_copy(uint32_t dst, const void* src) {
    if (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}

// Queries as the kernel below reads them, one of these per sequence and head: 32 GP bytes, for every group the word
// (0, multiple of 4 beyond its sum) and the word (0, what that has too much) as halves, then the scale in base 2.
// |sum| <= 4064: both are halves, and as they differ in sign a lowest value that is not finite gives NaN.
__host__ __device__ constexpr int p4_query_bytes(int gp) { return 40 * gp + 16; }

// A warp turns and quantises one query head: lane j holds dims 4 j .. 4 j + 3 of every 128. (In the attention kernel
// itself this took 7 of the first 10 us of every run, for the instructions of all forms of the rotation; here it runs
// while that kernel finds its runs and requests its first keys.)
__global__ void __launch_bounds__(128) paged4_query_kernel(PagedAttn4 a, int gp, bool wide_q, bool wide_rope, unsigned char* out) {
    griddep_wait();  // first: the next kernel reads lengths, tables and pages before it waits for this one
    griddep_launch();
    const long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, b = (int)(i / a.H), h = (int)(i - (long long)b * a.H);
    if (b >= a.kv.num_seqs) return;
    const int len = p4_len(a, b);
    if (len == 0) return;  // no one reads its queries
    const float* q = a.Q + (size_t)b * a.ldq + (size_t)h * a.hd;
    const int pos = a.rope.cos_t ? (a.rope_pos ? __ldg(a.rope_pos + b) : len - 1) : 0;
    float4 x[2];
    float amax = 0.0f;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int d = 128 * k + 4 * lane;
        x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (d < a.hd) x[k] = a.rope.cos_t ? turned4(q, d, a.rope, pos, wide_rope) : p4_load4(q + d, wide_q);
        amax = fmaxf(fmaxf(amax, fmaxf(fabsf(x[k].x), fabsf(x[k].y))), fmaxf(fabsf(x[k].z), fabsf(x[k].w)));
    }
    amax = warp_max(amax);
    const float inv = q8_inv(amax);
    unsigned char* const to = out + (size_t)i * p4_query_bytes(gp);
    uint32_t* const sums = reinterpret_cast<uint32_t*>(to + 32 * gp);
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const uint32_t w = (uint32_t)(q8_round(x[k].x, inv) & 255) | (uint32_t)(q8_round(x[k].y, inv) & 255) << 8 |
                           (uint32_t)(q8_round(x[k].z, inv) & 255) << 16 | (uint32_t)q8_round(x[k].w, inv) << 24;
        int sum = __dp4a((int)w, 0x01010101, 0);
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const int group = 4 * k + (lane >> 3);
        if (group >= gp) continue;
        reinterpret_cast<uint32_t*>(to)[32 * k + lane] = w;
        if ((lane & 7) == 0) {
            const int hi = sum >= 0 ? (sum & ~3) + 4 : -((-sum & ~3) + 4);
            sums[group] = (uint32_t)__half_as_ushort(__int2half_rn(hi)) << 16;
            sums[gp + group] = (uint32_t)__half_as_ushort(__int2half_rn(sum - hi)) << 16;
        }
    }
    if (lane == 0) reinterpret_cast<float*>(sums + 2 * gp)[0] = __fmul_rn(q8_scale(amax), __fmul_rn(a.scale, 1.44269504088896341f));
}

template <int GP, int HEADS, bool TMA>
__global__ void __launch_bounds__(P4Cfg<GP, HEADS, TMA>::WARPS * 32, 1)
    paged4_attention_kernel(PagedAttn4 a, PaPlan pl, PaWork work, P4Scores scores, const unsigned char* queries, int param_copy,
                            const __grid_constant__ P4Maps maps) {
    using G = P4Cfg<GP, HEADS, TMA>;
    constexpr int TK = G::TK, U = G::U, ST = G::ST, ROWS = G::ROWS, E = G::E, ND = 2 * GP, PW = G::PW, LW = PW / 4;
    extern __shared__ __align__(128) unsigned char p4_raw[];
    unsigned char* const p4_sm = TMA ? p4_raw + (-smem_u32(p4_raw) & 1023u) : p4_raw;
    __shared__ __align__(8) uint64_t s_bar[G::WARPS][ST];
    __shared__ PaShared<G> sh;
    const uint64_t policy = policy_evict_first();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int group = a.H / a.KV, hd = a.hd, groups = TMA ? GP : (hd + 31) >> 5;
    griddep_launch();
    unsigned char* const ring = p4_sm + warp * G::RING;
    const uint32_t ring_a = smem_u32(ring);
    if (TMA && lane == 0) {
        if (warp == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.k) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.v) : "memory");
        }
        for (int i = 0; i < ST; i++) mbar_init(&s_bar[warp][i], 1);
        mbar_fence_init();
    }
    // parameters behind the head's last group: no copy writes them
    if (groups < PW)
        for (int st = 0; st < ST; st++)
            for (int i = groups; i < PW; i++)
                for (int j = lane; j < TK; j += 32) {
                    reinterpret_cast<uint32_t*>(ring + st * G::STAGE + G::KPOFF)[PW * j + i] = 0u;
                    reinterpret_cast<uint32_t*>(ring + st * G::STAGE + G::VPOFF)[PW * j + i] = 0u;
                }
    const PaRun run = pa_start<G>(a, pl, sh, hd);
    const long long w0 = run.w0, u0 = run.u0;
    const bool joint = run.joint;
    const int step = run.step;
    int count = run.count;
    PaCursor cur = run.cur;
    long long item0 = run.item0;
    if (tid == 0) work.tail[blockIdx.x].ctas = 0;

    // copies: lane j looks up the pages of keys j and j + 32 of a unit one step before the unit's copies are issued
    PaCursor nx = cur;
    int issued = 0;  // units whose pages are looked up
    int pg[U], slot[U], h = -1;
    long long hoff = 0, hpoff = 0;  // of kv head h
    bool ok[U];
    unsigned counts[U];  // whether this lane's key counts, of the unit issued last in bit 0
#pragma unroll
    for (int u = 0; u < U; u++) counts[u] = 0u;
    auto lookup = [&] {
#pragma unroll
        for (int u = 0; u < U; u++) ok[u] = false;
        if (issued < count) {
            const int r = pa_row<G>(pl, nx), hn = pl.qblocks == 1 ? r : r / pl.qblocks;
            if (hn != h) {
                h = hn;
                if (!TMA) hoff = (long long)h * a.kv.p.head_stride;
                hpoff = (long long)h * a.kv.p.phead_stride;
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int pos = nx.t * TK + 32 * u + lane;
                if (pos < nx.len) {
                    const int idx = a.kv.by_page(pos);
                    slot[u] = pos - idx * a.kv.p.page_size;
                    pg[u] = __ldg(a.kv.table + (size_t)nx.b * a.kv.table_stride + idx);
                    ok[u] = true;
                }
            }
            pa_next<G>(a, pl, nx, step);
        }
        issued++;
    };
    constexpr int LPR = GP <= 2 ? 2 : GP <= 4 ? 4 : 8, RPI = 32 / LPR;  // lanes per row, rows per step
    const int cc = lane & (LPR - 1), cr = lane / LPR;
    // the unit that was looked up last: rows, and by lane j its keys' parameters
    auto issue = [&](int st) {
        unsigned bytes = 0u;
        uint64_t* const bar = &s_bar[warp][st];
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (ok[u] && (unsigned)pg[u] >= (unsigned)a.kv.p.num_pages) {
                p4_flag(a.kv, kPagedErrPage);
                ok[u] = false;
            }
            counts[u] = counts[u] << 1 | (ok[u] ? 1u : 0u);
            if (TMA) bytes += __popc(__ballot_sync(0xffffffffu, ok[u] && (lane & (pl.box - 1)) == 0)) * pl.box * 32 * GP;
        }
        if (TMA) {
            if (lane == 0) mbar_expect_tx(bar, bytes);
            __syncwarp();
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int key = 32 * u + lane;
            const uint32_t base = ring_a + st * G::STAGE;
            if (ok[u]) {
                const long long po =
                    (long long)pg[u] * a.kv.p.ppage_stride + (long long)slot[u] * a.kv.p.ppos_stride + hpoff;
                const uint32_t* const kp = reinterpret_cast<const uint32_t*>(a.kv.p.kp) + po;
                const uint32_t* const vp = reinterpret_cast<const uint32_t*>(a.kv.p.vp) + po;
                const uint32_t dst = base + G::KPOFF + 4 * PW * key;
                if (param_copy == 4 * GP && 4 * GP <= 16) {
                    p4_copy<(4 * GP <= 16 ? 4 * GP : 16)>(dst, kp);
                    p4_copy<(4 * GP <= 16 ? 4 * GP : 16)>(dst + (G::VPOFF - G::KPOFF), vp);
                } else if (GP == 8 && param_copy == 32) {
#pragma unroll
                    for (int i = 0; i < 8; i += 4) {
                        p4_copy<16>(dst + 4 * i, kp + i);
                        p4_copy<16>(dst + (G::VPOFF - G::KPOFF) + 4 * i, vp + i);
                    }
                } else {
                    for (int i = 0; i < groups; i++) {
                        p4_copy<4>(dst + 4 * i, kp + i);
                        p4_copy<4>(dst + (G::VPOFF - G::KPOFF) + 4 * i, vp + i);
                    }
                }
            }
            if constexpr (TMA) {
                if (ok[u] && (lane & (pl.box - 1)) == 0) {
                    pa_tensor_copy(base + key * G::PITCH, &maps.k, h, slot[u], pg[u], bar, policy);
                    pa_tensor_copy(base + G::VOFF + key * G::PITCH, &maps.v, h, slot[u], pg[u], bar, policy);
                }
            } else {
                const unsigned mask = __ballot_sync(0xffffffffu, ok[u]);
                const long long off =
                    ok[u] ? (long long)pg[u] * a.kv.p.page_stride + (long long)slot[u] * a.kv.p.pos_stride + hoff : 0LL;
#pragma unroll
                for (int i = 0; i < 32 / RPI; i++) {
                    const int row = i * RPI + cr;
                    const long long o = __shfl_sync(0xffffffffu, off, row) + 16 * cc;
                    if (cc < groups && ((mask >> row) & 1)) {
                        const uint32_t dst = base + (32 * u + row) * G::PITCH + 16 * cc;
                        pa_copy<16>(dst, a.kv.p.k + o, policy);
                        pa_copy<16>(dst + G::VOFF, a.kv.p.v + o, policy);
                    }
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    // lane (g, t): query head g (and g + 8) as B fragments, bytes 4 t .. 4 t + 3 of every 16, its sums over groups as
    // halves; of the results the heads 2 t, 2 t + 1 (and 8 more), for which it keeps the reference, its share of the
    // sum, the dims 2 g, 2 g + 1 of every 16 in units of 2^(eg - 15) of their group (the high 16 of a group 16 times
    // that), and the products with column g (and g + 8) of V's parameters: (step, low) of each group
    uint32_t qf[GP][E][2], qsum[E][2 * LW];
    float qsl[E][2], ref[E][2], l[E][2], o[ND][E][4], opar[E][2 * LW];
    int eg[GP];        // exponent field of V's units of each group
    uint32_t ug[GP];   // p4_units of it
    bool fresh = true, tail = false;  // tail: the run ends inside an item that it starts
    bool gave_up = false;
    int st = 0;
    uint32_t phase = 0u;
    if (count > 0) {
        lookup();
#pragma unroll 1
        for (int i = 0; i < (TMA ? ST : ST - 1); i++) {
            issue(i);
            lookup();
        }
    }
    griddep_wait();  // the queries

    for (int n = 0; n < count; n++) {
        if (fresh) {
            fresh = false;
            const int r = pa_row<G>(pl, cur), qb = r % pl.qblocks, kvh = r / pl.qblocks;
#pragma unroll
            for (int i = 0; i < GP; i++) {
                eg[i] = 0;
                ug[i] = p4_units(0);
            }
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int row = qb * ROWS + 8 * e + (HEADS <= 4 ? g & 3 : g), own = qb * ROWS + 8 * e + 2 * t;
                const unsigned char* const at = queries + ((size_t)cur.b * a.H + (size_t)kvh * group) * p4_query_bytes(GP);
                const uint32_t* const q = reinterpret_cast<const uint32_t*>(at + (size_t)row * p4_query_bytes(GP));
#pragma unroll
                for (int i = 0; i < 2 * GP; i++) qf[i >> 1][e][i & 1] = row < group ? __ldcg(q + 4 * i + t) : 0u;
#pragma unroll
                for (int i = 0; i < 2 * LW; i++) {
                    const int k = 4 * (i % LW) + t;
                    qsum[e][i] = row < group && k < GP ? __ldcg(q + 8 * GP + (i / LW) * GP + k) : 0u;
                }
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int head = HEADS <= 4 ? qb * ROWS + (2 * t + i & 3) : own + i;
                    qsl[e][i] = head < group ? __ldcg(reinterpret_cast<const float*>(at + (size_t)head * p4_query_bytes(GP) + 40 * GP)) : 0.0f;
                    ref[e][i] = kPaLow;
                    l[e][i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 2 * LW; i++) opar[e][i] = 0.0f;
#pragma unroll
                for (int d = 0; d < ND; d++) o[d][e][0] = o[d][e][1] = o[d][e][2] = o[d][e][3] = 0.0f;
            }
        }
        if constexpr (!TMA) {
            // the next unit's copies go to the stage that the last iteration read
            __syncwarp();
            issue(st == 0 ? ST - 1 : st - 1);
            lookup();
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
        __syncwarp();
        if constexpr (TMA)
            if (!pa_wait(&s_bar[warp][st], phase, a.kv.err)) gave_up = true;
        unsigned char* const sb = ring + st * G::STAGE;
        const uint32_t base = ring_a + st * G::STAGE;
        unsigned in[U];  // keys that count
        bool full = true;
#pragma unroll
        for (int u = 0; u < U; u++) {
            in[u] = __ballot_sync(0xffffffffu, (counts[u] >> (ST - 1)) & 1u);
            full &= in[u] == ~0u;
        }

        // lane j, its keys: V's steps in units of their group, laid out by group as the products read them
        bool apart = false;  // the unit's values do not fit units of any size
        float room;          // how far below the reference its keys may score: 2^4, or 2^8 of values within 2^4
        {
            uint32_t vw[U][PW];
            __half2 top = __float2half2_rn(0.0f), bottom = __float2half2_rn(2.0f);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const bool live = full || (in[u] >> lane & 1);
                uint32_t* const vrow = reinterpret_cast<uint32_t*>(sb + G::VPOFF) + PW * (32 * u + lane);
                if (!live)  // whatever the ring held
#pragma unroll
                    for (int i = 0; i < PW; i++) vrow[i] = 0u;
                p4_words(vrow, vw[u]);
#pragma unroll
                for (int i = 0; i < GP; i++) {
                    const __half2 x = __habs2(__hmul2_rn(p4_h2(vw[u][i]), p4_h2(ug[i])));
                    top = __hmax2_nan(top, x);
                    if (i < groups && live) bottom = __hmin2(bottom, x);
                }
            }
            const bool small = __hblt2(top, __float2half2_rn(2.0f));
            room = __all_sync(0xffffffffu, small && __low2float(bottom) >= 0x1p-4f) ? 8.0f : 4.0f;
            if (!__all_sync(0xffffffffu, small && __low2float(bottom) >= 0x1p-8f)) {  // other units for the groups that do not fit theirs
#pragma unroll
                for (int i = 0; i < GP; i++) {
                    auto all_fit = [&](int e1) {
                        bool y = true;
#pragma unroll
                        for (int u = 0; u < U; u++) y &= p4_fits(vw[u][i], e1) || !(in[u] >> lane & 1);
                        return __all_sync(0xffffffffu, y) != 0;
                    };
                    if (all_fit(eg[i])) continue;
                    uint32_t most = 0u;  // bits of the largest step, or of an eighth of the largest low
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        const uint32_t step = vw[u][i] & 0x7fffu, low = vw[u][i] >> 16 & 0x7fffu;
                        most = max(most, max(step, low > 0x0c00u ? low - 0x0c00u : low ? 1u : 0u));
                    }
                    most = __reduce_max_sync(0xffffffffu, most);
                    if (most == 0u) continue;  // zeros
                    const int e1 = min((int)(most >> 10), 30);
                    apart |= !all_fit(e1);
                    const float f = p4_pow2(eg[i] - e1);
                    eg[i] = e1;
                    ug[i] = p4_units(e1);
#pragma unroll
                    for (int e = 0; e < E; e++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            o[2 * i][e][j] *= f;
                            o[2 * i + 1][e][j] *= f;
                        }
                }
            }
            __half* const to = reinterpret_cast<__half*>(ring + G::SOFF) + 8 * ((lane & 7) >> 1) + 2 * (lane >> 3) + (lane & 1);
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int i = 0; i < GP; i++)
                    to[32 * (GP * u + i)] = __low2half(__hmul2_rn(p4_h2(vw[u][i]), p4_h2(ug[i])));
        }
        __syncwarp();

        // scores of keys 8 i + g and heads 2 t, + 1, in base 2: the parameters' products with (0, query sum) of each group,
        // then the groups' whole-number dots, which start at the bits of 1.5 * 2^23 (|dot| < 2^16), so an exact subtraction
        // makes them floats
        float s[4 * U][E][2];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t* const kp = reinterpret_cast<const uint32_t*>(sb + G::KPOFF) + 32 * PW * u;
            uint32_t par[LW][4];
#pragma unroll
            for (int i = 0; i < LW; i++) pa_ldsm(base + G::KPOFF + 4 * PW * (32 * u + lane) + 16 * i, par[i]);
            float acc[2][E][4];
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int e = 0; e < E; e++) {
                    if constexpr (LW == 1) {
                        const uint32_t pf[4] = {par[0][2 * m], par[0][2 * m + 1], par[0][2 * m], par[0][2 * m + 1]};
                        pa_mma_f16(pf, qsum[e], 0.0f, acc[m][e]);
                    } else {
                        const uint32_t pf[4] = {par[0][2 * m], par[0][2 * m + 1], par[1][2 * m], par[1][2 * m + 1]};
                        const uint32_t q0[2] = {qsum[e][0], qsum[e][1]}, q1[2] = {qsum[e][2], qsum[e][3]};
                        pa_mma_f16(pf, q0, 0.0f, acc[m][e]);
                        pa_mma_f16(pf, q1, acc[m][e]);
                    }
                }
#pragma unroll
            for (int i0 = 0; i0 < GP; i0 += 2) {
                uint32_t w[4][2];
#pragma unroll
                for (int i = 0; i < 4; i++) p4_words(kp + PW * (8 * i + g) + i0, w[i]);
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    uint32_t r[4];
                    pa_ldsm(base + G::at(32 * u + lane, i0 + k), r);
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        const uint32_t kf[4] = {r[2 * m] & 0x0F0F0F0Fu, r[2 * m + 1] & 0x0F0F0F0Fu,
                                                r[2 * m] >> 4 & 0x0F0F0F0Fu, r[2 * m + 1] >> 4 & 0x0F0F0F0Fu};
                        const float s0 = p4_step(w[2 * m][k]), s1 = p4_step(w[2 * m + 1][k]);
#pragma unroll
                        for (int e = 0; e < E; e++) {
                            int c[4];
                            pa_mma_s8(kf, qf[i0 + k][e], 0x4B400000, c);
#pragma unroll
                            for (int j = 0; j < 4; j += 2) {
                                float x = __int_as_float(c[j]), y = __int_as_float(c[j + 1]);
                                p4_add2(x, y, -12582912.0f, -12582912.0f);
                                p4_fma2(acc[m][e][j], acc[m][e][j + 1], j ? s1 : s0, j ? s1 : s0, x, y);
                            }
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < E; e++)
                {
                    s[4 * u + i][e][0] = acc[i >> 1][e][2 * (i & 1)];
                    s[4 * u + i][e][1] = acc[i >> 1][e][2 * (i & 1) + 1];
                    p4_mul2(s[4 * u + i][e][0], s[4 * u + i][e][1], qsl[e][0], qsl[e][1]);
                }
        }
        if (!full) {  // keys that do not count: -inf, whatever the ring held
#pragma unroll
            for (int i = 0; i < 4 * U; i++)
#pragma unroll
                for (int e = 0; e < E; e++)
#pragma unroll
                    for (int j = 0; j < 2; j++) s[i][e][j] = in[i >> 2] >> (8 * (i & 3) + g) & 1 ? s[i][e][j] : -INFINITY;
        }
        if (scores.s && (HEADS > 4 || t < 2)) {
            float* const to = scores.s + p4_score_at(scores, pl, cur.b, pa_row<G>(pl, cur), cur.t, TK * ROWS) + 2 * t;
#pragma unroll
            for (int i = 0; i < 4 * U; i++)
#pragma unroll
                for (int e = 0; e < E; e++)
                    *reinterpret_cast<float2*>(to + ROWS * (8 * i + g) + 8 * e) = make_float2(s[i][e][0], s[i][e][1]);
        }
        // the reference follows the maximum; a unit that scores far below it takes its weights 2^d up
        float top[E][2], down[E][2];  // down: 2^-d
        bool raise = false, near = true;
#pragma unroll
        for (int e = 0; e < E; e++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                float x = fmaxf(fmaxf(s[0][e][j], s[1][e][j]), fmaxf(s[2][e][j], s[3][e][j]));
                if (U > 1) {
                    constexpr int b = 4 * (U - 1);
                    x = fmaxf(x, fmaxf(fmaxf(s[b][e][j], s[b + 1][e][j]), fmaxf(s[b + 2][e][j], s[b + 3][e][j])));
                }
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                top[e][j] = x - kPaShift;
                down[e][j] = 1.0f;
                raise |= top[e][j] > ref[e][j];
                near &= top[e][j] > ref[e][j] - room;
            }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int e = 0; e < E; e++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float to = fmaxf(ref[e][j], top[e][j]), al = ex2(ref[e][j] - to);
                    ref[e][j] = to;
                    l[e][j] *= al;
#pragma unroll
                    for (int i = 0; i < LW; i++) opar[e][2 * i + j] *= al;
#pragma unroll
                    for (int d = 0; d < ND; d++) {
                        o[d][e][j] *= al;
                        o[d][e][2 + j] *= al;
                    }
                }
        }
#pragma unroll
        for (int i = 0; i < 4 * U; i++)
#pragma unroll
            for (int e = 0; e < E; e++) p4_add2(s[i][e][0], s[i][e][1], -ref[e][0], -ref[e][1]);
        if (!__all_sync(0xffffffffu, near))
#pragma unroll
            for (int e = 0; e < E; e++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    // (with no key, or behind all that fp32 holds, the weights stay as they are)
                    const float d = floorf(ref[e][j] - top[e][j]);
                    const bool up = d >= 4.0f && d <= 126.0f;
                    if (up) down[e][j] = p4_pow2(-(int)d);
#pragma unroll
                    for (int i = 0; i < 4 * U; i++) s[i][e][j] += up ? d : 0.0f;
                }
        if (!apart) {
            // weights as halves hi + lo, transposed: column g, keys 8 i + 2 t, + 1
            uint32_t hi[4 * U][E], lo[4 * U][E];
#pragma unroll
            for (int i = 0; i < 4 * U; i++)
#pragma unroll
                for (int e = 0; e < E; e++) {
                    float b0 = ex2(s[i][e][0]), b1 = ex2(s[i][e][1]);
                    p4_fma2(l[e][0], l[e][1], b0, b1, down[e][0], down[e][1]);
                    const uint32_t ph = pa_pack(b0, b1);
                    const float2 hf = __half22float2(p4_h2(ph ^ 0x80008000u));
                    p4_add2(b0, b1, hf.x, hf.y);
                    hi[i][e] = pa_transpose(ph);
                    lo[i][e] = pa_transpose(pa_pack(b0, b1));
                }
            // the parameters' share: rows are their columns
            {
                float c[E][4];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    uint32_t par[LW][4];
#pragma unroll
                    for (int i = 0; i < LW; i++) pa_ldsm_t(base + G::VPOFF + 4 * PW * (32 * u + lane) + 16 * i, par[i]);
#pragma unroll
                    for (int e = 0; e < E; e++)
#pragma unroll
                        for (int m = 0; m < 2; m++) {
                            const uint32_t pf[4] = {par[0][2 * m], LW > 1 ? par[LW - 1][2 * m] : 0u, par[0][2 * m + 1],
                                                    LW > 1 ? par[LW - 1][2 * m + 1] : 0u};
                            const int i = 4 * u + 2 * m;
                            const uint32_t h0 = hi[i][e], h1 = hi[i + 1][e], l0 = lo[i][e], l1 = lo[i + 1][e];
                            if (HEADS <= 4) {
                                const uint32_t b[2] = {g < 4 ? h0 : l0, g < 4 ? h1 : l1};
                                if (i == 0)
                                    pa_mma_f16(pf, b, 0.0f, c[e]);
                                else
                                    pa_mma_f16(pf, b, c[e]);
                            } else {
                                const uint32_t bl[2] = {l0, l1}, bh[2] = {h0, h1};
                                if (i == 0)
                                    pa_mma_f16(pf, bl, 0.0f, c[e]);
                                else
                                    pa_mma_f16(pf, bl, c[e]);
                                pa_mma_f16(pf, bh, c[e]);
                            }
                        }
                }
#pragma unroll
                for (int e = 0; e < E; e++)
#pragma unroll
                    for (int i = 0; i < 2 * LW; i++) opar[e][i] = __fmaf_rn(c[e][i], down[e][i & 1], opar[e][i]);
            }
            // P.V, a group at a time: V's numbers less 8 as halves (the high ones 16 times that), rows g dims 2 g,
            // rows g + 8 dims 2 g + 1 of 16; a weight times a step as halves: hi rounded, lo what that left and lo's share.
            // 4 heads fill 8 columns with their hi and lo halves
            uint32_t zl[4 * U];
            if (HEADS <= 4)
#pragma unroll
                for (int i = 0; i < 4 * U; i++) {
                    zl[i] = g < 4 ? 0u : hi[i][0] ^ 0x80008000u;
                    lo[i][0] = g < 4 ? 0u : lo[i][0];
                }
#pragma unroll
            for (int i0 = 0; i0 < GP; i0++) {
                float c[2][E][4];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    uint32_t r[4];
                    pa_ldsm_t(base + G::VOFF + G::at(32 * u + lane, i0), r);
                    const uint4 sv = *reinterpret_cast<const uint4*>(ring + G::SOFF + 64 * (GP * u + i0) + 16 * t);
                    const uint32_t sw[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        uint32_t bh[E][2], bl[E][2];
#pragma unroll
                        for (int e = 0; e < E; e++)
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                const int at = 4 * u + 2 * m + i;
                                const __half2 w = p4_h2(sw[2 * m + i]), ph = p4_h2(hi[at][e]), pw = p4_h2(lo[at][e]);
                                if (HEADS <= 4) {
                                    bh[e][i] = p4_u(__hfma2(pw, w, __hfma2(ph, w, __hmul2_rn(p4_h2(zl[at]), w))));
                                } else {
                                    const __half2 x = __hmul2_rn(ph, w);
                                    bh[e][i] = p4_u(x);
                                    bl[e][i] = p4_u(__hfma2(pw, w, __hfma2(ph, w, __hneg2(x))));
                                }
                            }
                        const uint32_t x0 = r[2 * m], x1 = r[2 * m + 1], y0 = x0 >> 8, y1 = x1 >> 8;
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const uint32_t vf[4] = {k ? p4_whole<true>(x0) : p4_whole<false>(x0), k ? p4_whole<true>(y0) : p4_whole<false>(y0),
                                                    k ? p4_whole<true>(x1) : p4_whole<false>(x1), k ? p4_whole<true>(y1) : p4_whole<false>(y1)};
#pragma unroll
                            for (int e = 0; e < E; e++) {
                                if (u == 0 && m == 0)
                                    pa_mma_f16(vf, bh[e], 0.0f, c[k][e]);
                                else
                                    pa_mma_f16(vf, bh[e], c[k][e]);
                                if (HEADS > 4) pa_mma_f16(vf, bl[e], c[k][e]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int e = 0; e < E; e++)
#pragma unroll
                        for (int j = 0; j < 4; j += 2)
                            p4_fma2(o[2 * i0 + k][e][j], o[2 * i0 + k][e][j + 1], c[k][e][j], c[k][e][j + 1], down[e][0], down[e][1]);
            }
        } else {
            // key by key in fp32: the weights lie over K's rows, from where every lane takes those of its heads
            float* const pw = reinterpret_cast<float*>(sb);  // [key][ROWS]
            static_assert(4 * 32 * ROWS <= TK * G::PITCH, "32 keys' weights fit K's rows");
#pragma unroll
            for (int u = 0; u < U; u++) {
                __syncwarp();  // K's rows are read, and the last keys' weights
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const float p0 = ex2(s[4 * u + i][e][0]) * down[e][0], p1 = ex2(s[4 * u + i][e][1]) * down[e][1];
                        p4_add2(l[e][0], l[e][1], p0, p1);
                        if (HEADS > 4 || t < 2)
                            *reinterpret_cast<float2*>(pw + ROWS * (8 * i + g) + 8 * e + 2 * t) = make_float2(p0, p1);
                    }
                __syncwarp();
#pragma unroll 1
                for (int k = 0; k < 32; k++) {
                    const unsigned char* const par = sb + G::VPOFF + 4 * PW * (32 * u + k);
                    float2 p[E];
#pragma unroll
                    for (int e = 0; e < E; e++)
                        p[e] = HEADS > 4 || t < 2 ? *reinterpret_cast<const float2*>(pw + ROWS * k + 8 * e + 2 * t)
                                                  : make_float2(0.0f, 0.0f);  // their heads are counted at t - 2
#pragma unroll
                    for (int i = 0; i < LW; i++) {
                        const float x = __half2float(reinterpret_cast<const __half*>(par)[8 * i + g]);
#pragma unroll
                        for (int e = 0; e < E; e++) {
                            opar[e][2 * i] = __fmaf_rn(p[e].x, x, opar[e][2 * i]);
                            opar[e][2 * i + 1] = __fmaf_rn(p[e].y, x, opar[e][2 * i + 1]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < GP; i++) {
                        const float step = p4_step(reinterpret_cast<const uint32_t*>(par)[i]) * p4_pow2(15 - eg[i]);
                        const int n2 = *reinterpret_cast<const unsigned short*>(sb + G::VOFF + G::at(32 * u + k, i) + 2 * g);
#pragma unroll
                        for (int c = 0; c < 2; c++) {  // the low and the high bits: 16 times their numbers
                            const float x = (float)(c ? (n2 & 0xF0) - 128 : (n2 & 15) - 8) * step;
                            const float y = (float)(c ? (n2 >> 8 & 0xF0) - 128 : (n2 >> 8 & 15) - 8) * step;
#pragma unroll
                            for (int e = 0; e < E; e++) {
                                o[2 * i + c][e][0] = __fmaf_rn(p[e].x, x, o[2 * i + c][e][0]);
                                o[2 * i + c][e][1] = __fmaf_rn(p[e].y, x, o[2 * i + c][e][1]);
                                o[2 * i + c][e][2] = __fmaf_rn(p[e].x, y, o[2 * i + c][e][2]);
                                o[2 * i + c][e][3] = __fmaf_rn(p[e].y, y, o[2 * i + c][e][3]);
                            }
                        }
                    }
                }
            }
            if (TMA) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // tensor copies write there next
            __syncwarp();
        }
        if constexpr (TMA) {
            // the stage is read: the unit ST ahead takes its place
            if (__any_sync(0xffffffffu, gave_up)) {
                count = n + 1;  // the run ends here
                gave_up = true;
            } else {
                issue(st);
                lookup();
            }
        }
        if (++st == ST) {
            st = 0;
            phase ^= 1u;
        }

        const bool item_end = cur.t == cur.nt - 1;
        if (n + 1 < count && (joint || !item_end)) {
            cur.t += step;
            continue;
        }
        // the end of an item or of the run: a parameter of V that is not finite makes all of its rows NaN
#pragma unroll
        for (int e = 0; e < E; e++) {
            float z[2] = {0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < 2; j++) {
#pragma unroll
                for (int i = 0; i < LW; i++) z[j] = __fmaf_rn(opar[e][2 * i + j], 0.0f, z[j]);
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) z[j] += __shfl_xor_sync(0xffffffffu, z[j], x);
            }
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const float f = __uint_as_float((uint32_t)(eg[d >> 1] - 15 + 127 - 4 * (d & 1)) << 23);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    // low + 8 step of the group's numbers
                    const float par = opar[e][2 * (d >> 3) + j];
                    const float x = __fmaf_rn(8.0f, __shfl_sync(0xffffffffu, par, 8 * (d >> 1 & 3) + t),
                                              __shfl_sync(0xffffffffu, par, 8 * (d >> 1 & 3) + 4 + t)) + z[j];
                    o[d][e][j] = __fmaf_rn(o[d][e][j], f, x);
                    o[d][e][2 + j] = __fmaf_rn(o[d][e][2 + j], f, x);
                }
            }
#pragma unroll
            for (int j = 0; j < 2; j++) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[e][j] += __shfl_xor_sync(0xffffffffu, l[e][j], x);
                l[e][j] += z[j];
            }
        }
        if (HEADS <= 4)  // lanes t and t + 2 hold the sums of hi and lo halves of the same heads
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int j = 0; j < 4; j++) o[d][0][j] += __shfl_xor_sync(0xffffffffu, o[d][0][j], 2);
        const bool from_start = item0 >= u0;
        if (joint ? run.alone : from_start && item_end) {
            pa_finish<G>(a, pl, work, cur, hd, o, ref, l);
        } else {
            if (joint) break;  // o, ref and l stay in registers
            tail = from_start;
            pa_store<G>(work.part + ((size_t)(w0 * pl.team + warp) * 2 + (from_start ? 1 : 0)) * G::PART, true, o, ref, l);
        }
        if (n + 1 < count) {
            item0 += cur.nt;
            pa_next<G>(a, pl, cur, 1);
            fresh = true;
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (TMA && gave_up)  // the copies that are still on their way write to this CTA's memory
        for (int i = 0; i < ST; i++) {
            pa_wait(&s_bar[warp][st], phase, a.kv.err);
            if (++st == ST) {
                st = 0;
                phase ^= 1u;
            }
        }
    pa_end<G>(a, pl, work, sh, run, count, cur, item0, tail, p4_sm, hd, o, ref, l);
}

// The weights of the scores that the kernel above left, added to their keys' mass: kP4MassKeys keys of a thread in flight.
constexpr int kP4MassThreads = 128, kP4MassKeys = 4;
template <int ROWS>
__global__ void __launch_bounds__(kP4MassThreads) paged4_mass_kernel(PagedAttn4 a, PaPlan pl, PaWork work, P4Scores scores) {
    griddep_wait();
    const int b = blockIdx.x / a.KV, kvh = blockIdx.x - b * a.KV, group = a.H / a.KV;
    const int len = p4_len(a, b);
    const float2* const stat = work.stat + (size_t)b * a.H + (size_t)kvh * group;
    float2 ri[ROWS];
    auto stats = [&](int qb) {
#pragma unroll
        for (int i = 0; i < ROWS; i++) ri[i] = qb * ROWS + i < group ? __ldcg(stat + qb * ROWS + i) : make_float2(0.0f, 0.0f);
    };
    stats(0);
    for (long long j0 = (long long)blockIdx.y * kP4MassThreads * kP4MassKeys + threadIdx.x; j0 < len;
         j0 += (long long)gridDim.y * kP4MassThreads * kP4MassKeys) {
        int slot[kP4MassKeys], page[kP4MassKeys];
        float sum[kP4MassKeys];
#pragma unroll
        for (int k = 0; k < kP4MassKeys; k++) {
            const long long j = j0 + k * kP4MassThreads;
            sum[k] = 0.0f;
            page[k] = j < len ? p4_entry(a.kv, b, (int)j, &slot[k]) : -1;
        }
        for (int qb = 0; qb < pl.qblocks; qb++) {
            const float* s = scores.s + p4_score_at(scores, pl, b, kvh * pl.qblocks + qb, (int)j0, ROWS);
            float4 x[kP4MassKeys][ROWS / 4];
#pragma unroll
            for (int k = 0; k < kP4MassKeys; k++)
#pragma unroll
                for (int i = 0; i < ROWS / 4; i++)
                    x[k][i] = page[k] != -1 ? __ldcg(reinterpret_cast<const float4*>(s + (size_t)k * kP4MassThreads * ROWS) + i)
                                            : make_float4(0.f, 0.f, 0.f, 0.f);
            if (pl.qblocks > 1) stats(qb);
#pragma unroll
            for (int k = 0; k < kP4MassKeys; k++)
#pragma unroll
                for (int i = 0; i < ROWS; i += 4) {
                    // rows behind the last head have no stat
                    const float4 v = x[k][i / 4];
                    const int left = group - qb * ROWS - i;
                    if (left > 0) sum[k] += ex2(v.x - ri[i].x) * ri[i].y;
                    if (left > 1) sum[k] += ex2(v.y - ri[i + 1].x) * ri[i + 1].y;
                    if (left > 2) sum[k] += ex2(v.z - ri[i + 2].x) * ri[i + 2].y;
                    if (left > 3) sum[k] += ex2(v.w - ri[i + 3].x) * ri[i + 3].y;
                }
        }
#pragma unroll
        for (int k = 0; k < kP4MassKeys; k++)
            if (page[k] != -1 && p4_valid(a.kv, page[k]))
                atomicAdd(a.kv.p.mass + p4_moff(a.kv.p, page[k], slot[k], kvh), sum[k]);
    }
}

size_t align16(size_t n) { return (n + 15) / 16 * 16; }

// The workspace of one call: tails, parts, queries, and where weights are gathered stat and scores.
template <int GP, int HEADS, bool TMA>
size_t p4_work(int ctas, int seqs, int H, int KV, int capacity, unsigned char* base, PaWork* w, P4Scores* sc,
               unsigned char** queries) {
    using G = P4Cfg<GP, HEADS, TMA>;
    const int qblocks = (H / KV + HEADS - 1) / HEADS;
    const size_t parts = align16(ctas * sizeof(PaTail));
    const size_t query = align16(parts + (size_t)ctas * G::WARPS * 2 * G::PART * sizeof(float));
    const size_t stat = align16(query + (size_t)seqs * H * p4_query_bytes(GP));
    const size_t score = align16(stat + (capacity ? (size_t)seqs * H * sizeof(float2) : 0));
    const long long keys = ((long long)capacity + G::TK - 1) / G::TK * G::TK * HEADS;
    if (base) {
        *w = PaWork{reinterpret_cast<PaTail*>(base), reinterpret_cast<float*>(base + parts),
                    capacity ? reinterpret_cast<float2*>(base + stat) : nullptr};
        *queries = base + query;
        *sc = P4Scores{capacity ? reinterpret_cast<float*>(base + score) : nullptr, keys};
    }
    return score + (size_t)seqs * KV * qblocks * keys * sizeof(float);
}

// Map of a cache array as [page][slot][kv head][byte], boxes of `box` slots of one head.
int p4_map(CUtensorMap* m, uint8_t* base, const PagedAttn4& a, int row, int box) {
    void* fn = nullptr;
    if (int e = tensor_map_encoder(&fn)) return e;
    const jyc_kv_pages_q4& p = a.kv.p;
    const cuuint64_t dims[4] = {(cuuint64_t)row, (cuuint64_t)a.KV, (cuuint64_t)p.page_size, (cuuint64_t)p.num_pages};
    // the stride of a dimension of one entry is not used, but has to be one
    const cuuint64_t strides[3] = {(cuuint64_t)(a.KV > 1 ? p.head_stride : row),
                                   (cuuint64_t)(p.page_size > 1 ? p.pos_stride : row),
                                   (cuuint64_t)(p.num_pages > 1 ? p.page_stride : row)};
    const cuuint32_t boxes[4] = {(cuuint32_t)row, 1, (cuuint32_t)box, 1}, step[4] = {1, 1, 1, 1};
    const CUresult r = reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(fn)(
        m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, base, dims, strides, boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
        row == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return cuda_fail(cudaErrorInvalidValue, "cuTensorMapEncodeTiled");
    return JYC_OK;
}

// Tensor copies need rows of 32 or 64 bytes, strides below 2^40, and pages that a unit of 32 keys fills or that fill half
// of one (smaller pages would need a copy each for few rows).
bool p4_tensor_copies(const PagedAttn4& a) {
    const jyc_kv_pages_q4& p = a.kv.p;
    const int groups = (a.hd + 31) / 32;
    const long long far = std::max(p.page_stride, std::max(p.pos_stride, p.head_stride));
    const bool nonzero = (p.head_stride > 0 || a.KV == 1) && p.pos_stride > 0 && (p.page_stride > 0 || p.num_pages == 1);
    return nonzero && far < (1LL << 40) && (groups == 2 || groups == 4) && (p.page_size % 32 == 0 || p.page_size == 16);
}

template <int GP, int HEADS, bool TMA>
int p4_launch(const PagedAttn4& a, PaPlan pl, int sms, void* work, cudaStream_t s) {
    using G = P4Cfg<GP, HEADS, TMA>;
    if (int e = max_dynamic_smem(reinterpret_cast<const void*>(paged4_attention_kernel<GP, HEADS, TMA>), G::SMEM)) return e;
    const int capacity = a.kv.table_stride * a.kv.p.page_size, groups = (a.hd + 31) / 32;
    const long long tiles = ((long long)capacity + G::TK - 1) / G::TK;
    // teams of as many neighbouring kv heads as the warps hold evenly: their rows lie side by side where pages hold
    // positions first (5 and 7 heads share no divisor with the warps: 78 and 81 us, 68 with 6 or 8 of as many keys in all)
    pl.team = std::gcd(pl.units_row, (int)G::WARPS);
    pl.units_row /= pl.team;
    const long long items = (long long)a.kv.num_seqs * pl.units_row;
    // no more CTAs than the longest possible lengths have units for
    const long long units = tiles >= (1LL << 31) / items ? 1LL << 31 : items * tiles, few = std::max(1, kPaFewWarps / pl.team);
    const int ctas = (int)std::max(1LL, std::min((long long)sms, (units + few - 1) / few));
    pl.tk = G::TK;
    const jyc_kv_pages_q4& p = a.kv.p;
    P4Maps maps{};
    if (TMA) {
        pl.box = std::min(p.page_size, 32);
        if (int e = p4_map(&maps.k, p.k, a, 16 * GP, pl.box)) return e;
        if (int e = p4_map(&maps.v, p.v, a, 16 * GP, pl.box)) return e;
    }
    PaWork w;
    P4Scores sc;
    unsigned char* queries;
    p4_work<GP, HEADS, TMA>(sms, a.kv.num_seqs, a.H, a.KV, p.mass ? capacity : 0, static_cast<unsigned char*>(work), &w, &sc,
                            &queries);
    const long long rows = (long long)a.kv.num_seqs * a.H;
    if (int e = launch_follow(paged4_query_kernel, dim3((unsigned)((rows + 3) / 4)), 128, 0, s, a, GP, pl.wide_q, pl.wide_rope, queries)) return e;
    // a key's parameters by one copy where their alignment allows it, else word by word
    const uintptr_t at = (uintptr_t)p.kp | (uintptr_t)p.vp | (uintptr_t)(4 * (p.ppage_stride | p.ppos_stride | p.phead_stride));
    const int copy = groups == GP && at % (4 * GP) == 0 ? 4 * GP : 4;
    if (int e = launch_follow(paged4_attention_kernel<GP, HEADS, TMA>, dim3(ctas), G::WARPS * 32, G::SMEM, s, a, pl, w, sc,
                          (const unsigned char*)queries, copy, maps))
        return e;
    if (tiles > 1)  // else an item is one unit: none is split
        if (int e = launch_follow(paged_join_wide_kernel<G>, dim3(ctas, (G::ROWS * pl.team + pa_wide_rows<G>(pl.team) - 1) / pa_wide_rows<G>(pl.team)), kPaWideThreads, 0, s, a, pl, w)) return e;
    if (!sc.s) return JYC_OK;
    const long long heads = (long long)a.kv.num_seqs * a.KV, most = ((long long)capacity + kP4MassThreads * kP4MassKeys - 1) / (kP4MassThreads * kP4MassKeys);
    const unsigned chunks = (unsigned)std::min({most, (32LL * sms + heads - 1) / heads, 65535LL});
    return launch_follow(paged4_mass_kernel<G::ROWS>, dim3((unsigned)heads, chunks), kP4MassThreads, 0, s, a, pl, w, sc);
}

// The instantiation of a shape: groups and query heads per unit rounded up.
#define P4_HEADS(F, GP, TMA, ...) \
    return R <= 4 ? F<GP, 4, TMA>(__VA_ARGS__) : R <= 8 ? F<GP, 8, TMA>(__VA_ARGS__) : F<GP, 16, TMA>(__VA_ARGS__)
#define P4_CASES(F, TMA, ...)                                \
    do {                                                     \
        const int R = H / KV;                                \
        if (hd <= 64) P4_HEADS(F, 2, TMA, __VA_ARGS__);      \
        if (hd <= 128) P4_HEADS(F, 4, TMA, __VA_ARGS__);     \
        if (hd <= 192) P4_HEADS(F, 6, false, __VA_ARGS__);   \
        P4_HEADS(F, 8, false, __VA_ARGS__);                  \
    } while (0)

// ---------------------------------------------------------------------------
// Eviction: a cluster finds which rows a kv head of a sequence keeps, then groups
// of lanes copy them.
//
// Select: the border among the masses' order keys (the `want`-th largest) digit by
// digit, 8 bits each: each CTA counts the digits of its slice of the positions in
// shared memory, all CTAs of the cluster add up all counts and find the same digit. Then
// kept positions are counted slice by slice and warp by warp, and written in their order.
// Keys of slices up to kEvSpan positions stay in shared memory (131072 positions of one
// sequence: 8 CTAs a head), those of longer ones are read again for each digit (10
// sequences of 8 heads: 44 us at 24000 positions, 89 at 25500). Masses
// differ little in their first digit: each lane has counts of its own. (Digits of 11 bits
// need one pass less, but 2048 counts to clear, add up and exchange: for 131072 positions 40 us against 33.)
constexpr int kEvThreads = 1024, kEvWarps = kEvThreads / 32, kEvSpan = 24576;
constexpr int kEvBins = 256, kEvDigits = 4, kEvMaxCluster = 8;
constexpr int kEvSmem = ((32 + kEvDigits) * kEvBins + kEvSpan) * 4;

// larger mass -> larger key; NaN below every number, -0 as 0
__device__ __forceinline__ uint32_t ev_key(float m) { return f32_order_key(m + 0.0f); }
__device__ __forceinline__ void ev_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int ev_far(const int* p, int rank) {
    uint32_t at;
    int v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

__global__ void __launch_bounds__(kEvThreads, 1) paged4_select_kernel(PagedEvict4 e, int ctas) {
    extern __shared__ int ev_sm[];
    int* const counts = ev_sm;                // [bin][lane]
    int* const sums = ev_sm + 32 * kEvBins;   // [digit][bin]: this CTA's
    uint32_t* const keys = reinterpret_cast<uint32_t*>(ev_sm + (32 + kEvDigits) * kEvBins);
    __shared__ int s_warp[kEvWarps], s_digit, s_above, s_count[2], s_more[kEvWarps], s_equal[kEvWarps];
    griddep_wait();
    griddep_launch();
    const int rank = blockIdx.x % ctas, item = blockIdx.x / ctas, b = item / e.KV, h = item - b * e.KV;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int len = max(e.lens[b], 0);
    const int cap = e.kv.table_stride * e.kv.p.page_size;
    if (len > cap) {
        p4_flag(e.kv, kPagedErrPos);
        len = cap;
    }
    int* kept = e.kept + (size_t)item * e.budget;
    if (h == 0 && rank == 0 && tid == 0) e.new_lens[b] = min(len, e.budget);
    if (len <= e.budget) {  // the whole cluster
        for (int i = rank * kEvThreads + tid; i < e.budget; i += ctas * kEvThreads) kept[i] = i < len ? i : -1;
        return;
    }
    const int old = len - e.recent, want = e.budget - e.recent;  // want < old
    for (int i = rank * kEvThreads + tid; i < e.recent; i += ctas * kEvThreads) kept[want + i] = old + i;
    if (want == 0) return;  // the whole cluster
    // this CTA's slice, and this warp's part of it: whole 32s of positions
    const int slice = (old + ctas - 1) / ctas, from = min(old, rank * slice), size = min(old, from + slice) - from;
    const int seg = (size + kEvThreads - 1) / kEvThreads * 32, w0 = min(size, warp * seg), w1 = min(size, w0 + seg);
    const bool cached = size <= kEvSpan;
    auto fetch = [&](int i) {
        int slot;
        const int page = p4_entry(e.kv, b, from + i, &slot);
        return p4_valid(e.kv, page) ? ev_key(e.kv.p.mass[p4_moff(e.kv.p, page, slot, h)]) : 0u;
    };
    if (cached) {
#pragma unroll 8
        for (int i = w0 + lane; i < w1; i += 32) keys[i] = fetch(i);
    }
    auto key = [&](int i) { return cached ? keys[i] : fetch(i); };
    uint32_t border = 0u;
    int left = want;  // of those that share the border's digits, how many are kept
#pragma unroll 1
    for (int d = 0; d < kEvDigits; d++) {
        const int shift = 24 - 8 * d;
        for (int i = tid; i < 32 * kEvBins / 4; i += kEvThreads) reinterpret_cast<int4*>(counts)[i] = make_int4(0, 0, 0, 0);
        __syncthreads();
#pragma unroll 4
        for (int i = w0 + lane; i < w1; i += 32) {
            const uint32_t k = key(i);
            if (d == 0 || (k ^ border) >> (shift + 8) == 0) atomicAdd(&counts[(k >> shift & (kEvBins - 1)) * 32 + lane], 1);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEvBins / kEvWarps; i++) {
            const int bin = warp * (kEvBins / kEvWarps) + i, n = __reduce_add_sync(0xffffffffu, counts[bin * 32 + lane]);
            if (lane == 0) sums[d * kEvBins + bin] = n;
        }
        __syncwarp();
        if (ctas > 1)
            ev_cluster_sync();
        else
            __syncthreads();
        // this thread's bin over all CTAs, all of their counts in flight at once, and a suffix sum over the bins
        int mine = 0;
        if (tid < kEvBins) {
            int far[kEvMaxCluster];
#pragma unroll
            for (int r = 0; r < kEvMaxCluster; r++) {
                far[r] = 0;
                if (r < ctas) far[r] = r == rank ? sums[d * kEvBins + tid] : ev_far(sums + d * kEvBins + tid, r);
            }
#pragma unroll
            for (int r = 0; r < kEvMaxCluster; r++) mine += far[r];
        }
        int above = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_down_sync(0xffffffffu, above, o);
            if (lane + o < 32) above += x;
        }
        if (lane == 0) s_warp[warp] = above;
        __syncthreads();
        above -= mine;
#pragma unroll
        for (int w = 1; w < kEvBins / 32; w++)
            if (w > warp) above += s_warp[w];
        if (tid < kEvBins && above < left && above + mine >= left) {  // one thread of the CTA
            s_digit = tid;
            s_above = above;
        }
        __syncthreads();
        border |= (uint32_t)s_digit << shift;
        left -= s_above;
    }
    // rows above the border and at it: of this warp, of the warps and CTAs before it
    int more = 0, equal = 0;
#pragma unroll 4
    for (int i = w0 + lane; i < w1; i += 32) {
        const uint32_t k = key(i);
        more += k > border;
        equal += k == border;
    }
    more = __reduce_add_sync(0xffffffffu, more);
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) {
        s_more[warp] = more;
        s_equal[warp] = equal;
    }
    __syncthreads();
    if (warp == 0) {
        const int a = __reduce_add_sync(0xffffffffu, s_more[lane]), c = __reduce_add_sync(0xffffffffu, s_equal[lane]);
        if (lane == 0) {
            s_count[0] = a;
            s_count[1] = c;
        }
    }
    int out = __reduce_add_sync(0xffffffffu, lane < warp ? s_more[lane] : 0);
    int ties = __reduce_add_sync(0xffffffffu, lane < warp ? s_equal[lane] : 0);
    if (ctas > 1) {
        __syncwarp();
        ev_cluster_sync();
        out += __reduce_add_sync(0xffffffffu, lane < rank ? ev_far(&s_count[0], lane) : 0);
        ties += __reduce_add_sync(0xffffffffu, lane < rank ? ev_far(&s_count[1], lane) : 0);
    }
    // of rows at the border the first `left` in order are kept
    out += min(ties, left);
#pragma unroll 4
    for (int i0 = w0; i0 < w1; i0 += 32) {
        const int i = i0 + lane;
        const uint32_t k = i < w1 ? key(i) : 0u;
        const bool tie = i < w1 && k == border;
        const unsigned t = __ballot_sync(0xffffffffu, tie), below = (1u << lane) - 1u;
        const bool keep = tie ? ties + __popc(t & below) < left : i < w1 && k > border;
        const unsigned m = __ballot_sync(0xffffffffu, keep);
        if (keep) kept[out + __popc(m & below)] = from + i;
        ties += __popc(t);
        out += __popc(m);
    }
    __syncwarp();
    if (ctas > 1) ev_cluster_sync();  // no CTA's memory goes while another one reads it
}

// A row is copied by as many lanes as it has 16-byte chunks (rounded up to a power of two), each with one chunk of K and
// one of V, the parameters word by word among them; kMvRows rows of a thread in flight.
constexpr int kMvThreads = 256, kMvRows = 2;
template <int LANES>
__global__ void __launch_bounds__(kMvThreads) paged4_move_kernel(PagedEvict4 e, FastDiv by_budget, FastDiv by_kv,
                                                                 FastDiv by_new_page) {
    constexpr int SIDE = kMvThreads / LANES;
    griddep_wait();
    const int sub = threadIdx.x & (LANES - 1), groups = (e.hd + 31) >> 5, total = e.kv.num_seqs * e.KV * e.budget;
    const jyc_kv_pages_q4& p = e.kv.p;
    const int w0 = blockIdx.x * (SIDE * kMvRows) + threadIdx.x / LANES;
    int from[kMvRows], b[kMvRows], h[kMvRows], to[kMvRows];
#pragma unroll
    for (int i = 0; i < kMvRows; i++) {
        const int w = w0 + i * SIDE;
        from[i] = w < total ? __ldcg(e.kept + w) : -1;
        const int item = by_budget(w);
        to[i] = w - item * e.budget;
        b[i] = by_kv(item);
        h[i] = item - b[i] * e.KV;
    }
    int sp[kMvRows], ss[kMvRows], dp[kMvRows], ds[kMvRows];
#pragma unroll
    for (int i = 0; i < kMvRows; i++) {
        sp[i] = dp[i] = -1;
        if (from[i] < 0) continue;
        sp[i] = p4_entry(e.kv, b[i], from[i], &ss[i]);
        const int idx = by_new_page(to[i]);
        ds[i] = to[i] - idx * p.page_size;
        dp[i] = __ldg(e.new_table + (size_t)b[i] * e.new_stride + idx);
    }
    uint4 k[kMvRows], v[kMvRows];
    uint32_t kp[kMvRows], vp[kMvRows];
    float m[kMvRows];
    bool ok[kMvRows];
#pragma unroll
    for (int i = 0; i < kMvRows; i++) {
        ok[i] = from[i] >= 0 && p4_valid(e.kv, sp[i]);
        if (from[i] >= 0 && (dp[i] < 0 || dp[i] >= p.num_pages)) {
            p4_flag(e.kv, kPagedErrPage);
            ok[i] = false;
        }
        if (!ok[i] || sub >= groups) continue;
        const size_t so = p4_off(p, sp[i], ss[i], h[i]) + 16 * sub, sq = p4_poff(p, sp[i], ss[i], h[i]) + sub;
        k[i] = *reinterpret_cast<const uint4*>(p.k + so);
        v[i] = *reinterpret_cast<const uint4*>(p.v + so);
        kp[i] = reinterpret_cast<const uint32_t*>(p.kp)[sq];
        vp[i] = reinterpret_cast<const uint32_t*>(p.vp)[sq];
        if (sub == 0) m[i] = p.mass[p4_moff(p, sp[i], ss[i], h[i])];
    }
#pragma unroll
    for (int i = 0; i < kMvRows; i++) {
        if (!ok[i] || sub >= groups) continue;
        const size_t to_ = p4_off(p, dp[i], ds[i], h[i]) + 16 * sub, dq = p4_poff(p, dp[i], ds[i], h[i]) + sub;
        *reinterpret_cast<uint4*>(p.k + to_) = k[i];
        *reinterpret_cast<uint4*>(p.v + to_) = v[i];
        reinterpret_cast<uint32_t*>(p.kp)[dq] = kp[i];
        reinterpret_cast<uint32_t*>(p.vp)[dq] = vp[i];
        if (sub == 0) p.mass[p4_moff(p, dp[i], ds[i], h[i])] = m[i];
    }
}

// The cache of rows r0, r0 + 1, ... when a row is its own sequence.
PagedKV4 shifted(PagedKV4 kv, const int* row_seq, int r0) {
    if (!row_seq) {
        kv.table += (size_t)r0 * kv.table_stride;
        kv.num_seqs -= r0;
    }
    return kv;
}

// Rows in launches of fewer than 2^30 warps of `per` heads. f(first row, rows, CTAs, warps that share K or V of a row).
template <class F>
int row_launches(int rows, int KV, int per, F f) {
    const int chunks = (KV + per - 1) / per, most = std::max(1, (1 << 30) / (2 * chunks)), warps = kP4Threads / 32;
    for (int r0 = 0; r0 < rows; r0 += most) {
        const int n = std::min(most, rows - r0);
        if (int e = f(r0, n, (unsigned)(((long long)n * 2 * chunks + warps - 1) / warps), chunks)) return e;
        if (rows - r0 <= most) break;
    }
    return JYC_OK;
}

template <int LANES, int UNITS>
auto append_of(int mode) {
    return mode == P4_PLAIN    ? paged4_append_kernel<LANES, UNITS, P4_PLAIN>
           : mode == P4_PAIRS  ? paged4_append_kernel<LANES, UNITS, P4_PAIRS>
           : mode == P4_HALVES ? paged4_append_kernel<LANES, UNITS, P4_HALVES>
                               : paged4_append_kernel<LANES, UNITS, P4_ODD>;
}

}  // namespace

int launch_paged4_append(const float* K, const float* V, int ld, int rows, int KV, int hd, const int* row_seq,
                         const int* row_pos, const int* rope_pos, const PagedKV4& kv, const RopeView& rope,
                         cudaStream_t s) {
    const bool vec = aligned16(K, ld) && aligned16(V, ld), wide = vec && rope_wide(rope);
    const int lanes = hd <= 32 ? 4 : hd <= 64 ? 8 : hd <= 128 ? 16 : 32, side = 32 / lanes;
    // four blocks of heads a warp where the rows have them and fill the SMs so: less bookkeeping a head; one otherwise
    // (with the read-back, as then measured: 16384 rows of 8 x 128 75 us, 83 with one; 8 rows 13 us with either)
    const bool many = KV > 2 * side && (long long)rows * KV >= 64LL * sm_count();
    const int mode = !rope.cos_t ? P4_PLAIN : !wide ? P4_ODD : rope.halves ? P4_HALVES : P4_PAIRS;
    const auto kernel = many ? (lanes == 4    ? append_of<4, 4>(mode)
                                : lanes == 8  ? append_of<8, 4>(mode)
                                : lanes == 16 ? append_of<16, 4>(mode)
                                              : append_of<32, 4>(mode))
                             : (lanes == 4    ? append_of<4, 1>(mode)
                                : lanes == 8  ? append_of<8, 1>(mode)
                                : lanes == 16 ? append_of<16, 1>(mode)
                                              : append_of<32, 1>(mode));
    return row_launches(rows, KV, (many ? 4 : 1) * side, [&](int r0, int n, unsigned grid, int chunks) {
        return launch_follow(kernel, dim3(grid), kP4Threads, 0, s, K + (size_t)r0 * ld, V + (size_t)r0 * ld, ld, n, KV, hd,
                             row_seq ? row_seq + r0 : nullptr, row_pos + r0, rope_pos ? rope_pos + r0 : nullptr,
                             shifted(kv, row_seq, r0), rope, chunks, fast_div(2 * chunks), vec);
    });
}

int launch_paged4_read(float* K, float* V, int ld, int rows, int KV, int hd, const int* row_seq, const int* row_pos,
                       const PagedKV4& kv, cudaStream_t s) {
    const bool vec = aligned16(K, ld) && aligned16(V, ld);
    const auto kernel = hd <= 32    ? paged4_read_kernel<8, 1>
                        : hd <= 64  ? paged4_read_kernel<16, 1>
                        : hd <= 128 ? paged4_read_kernel<32, 1>
                                    : paged4_read_kernel<32, 2>;
    return row_launches(rows, KV, kP4Units * (32 / (hd <= 32 ? 8 : hd <= 64 ? 16 : 32)), [&](int r0, int n, unsigned grid, int chunks) {
        return launch_follow(kernel, dim3(grid), kP4Threads, 0, s, K + (size_t)r0 * ld, V + (size_t)r0 * ld, ld, n, KV, hd,
                             row_seq ? row_seq + r0 : nullptr, row_pos + r0, shifted(kv, row_seq, r0), chunks,
                             fast_div(2 * chunks), vec);
    });
}

template <int GP, int HEADS, bool TMA>
static size_t p4_workspace(int sms, int seqs, int H, int KV, int capacity) {
    return p4_work<GP, HEADS, TMA>(sms, seqs, H, KV, capacity, nullptr, nullptr, nullptr, nullptr);
}

size_t paged4_attention_workspace(int seqs, int H, int KV, int hd, int capacity) {
    const int sms = std::min(sm_count(), kPaMaxCtas);
    if (sms == 0) return 0;
    P4_CASES(p4_workspace, false, sms, seqs, H, KV, capacity);  // the same with tensor copies
}

int launch_paged4_attention(const PagedAttn4& a, void* work, cudaStream_t s) {
    const int H = a.H, KV = a.KV, hd = a.hd, sms = std::min(sm_count(), kPaMaxCtas);
    PaPlan pl{};
    pl.qblocks = H / KV > 8 ? (H / KV + 15) / 16 : 1;
    pl.units_row = KV * pl.qblocks;
    pl.wide_q = aligned16(a.Q, a.ldq);
    pl.wide_rope = pl.wide_q && rope_wide(a.rope);
    if (p4_tensor_copies(a)) P4_CASES(p4_launch, true, a, pl, sms, work, s);
    P4_CASES(p4_launch, false, a, pl, sms, work, s);
}

int launch_paged4_evict(const PagedEvict4& e, cudaStream_t s) {
    if (int r = max_dynamic_smem(reinterpret_cast<const void*>(paged4_select_kernel), kEvSmem)) return r;
    const int items = e.kv.num_seqs * e.KV, sms = sm_count();
    const long long capacity = (long long)e.kv.table_stride * e.kv.p.page_size;
    // CTAs of a head: while the SMs hold them all and each has a few thousand positions
    int ctas = 1;
    while (ctas < kEvMaxCluster && (long long)items * ctas * 2 <= sms && capacity >= 4096LL * ctas) ctas *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)items * ctas);
    cfg.blockDim = dim3(kEvThreads);
    cfg.dynamicSmemBytes = kEvSmem;
    cfg.stream = s;
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = ctas;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    JYC_CUDA(cudaLaunchKernelEx(&cfg, paged4_select_kernel, e, ctas));
    JYC_LAUNCHED();
    const int groups = (e.hd + 31) / 32, lanes = groups <= 1 ? 1 : groups <= 2 ? 2 : groups <= 4 ? 4 : 8;
    const long long rows = (long long)items * e.budget, per = (long long)kMvThreads / lanes * kMvRows;
    const auto kernel = lanes == 1 ? paged4_move_kernel<1> : lanes == 2 ? paged4_move_kernel<2> : lanes == 4 ? paged4_move_kernel<4> : paged4_move_kernel<8>;
    return launch_follow(kernel, dim3((unsigned)((rows + per - 1) / per)), kMvThreads, 0, s, e, fast_div(e.budget), fast_div(e.KV),
                     e.kv.by_page);
}

}  // namespace jyc
