// paged.cu — int8 K/V cache in pages: rows are quantised as they are written
// (kv_pack_q8's rule, libs/model_libs/attention/attention_q8.h:20-37), read
// back as fp32, and attended over by one new token per sequence (the score,
// softmax and P.V of attention_q8.h:38-184).
#include "paged.cuh"
#include "ptx.cuh"

#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <mutex>

namespace jyc {

// Error word of the paged operators (kPagedErr* bits), apart from the decode
// kernel's own, which ends that kernel's waits.
__device__ int g_paged_err;

int* paged_error_word() {
    int* p = nullptr;
    if (cudaGetSymbolAddress(reinterpret_cast<void**>(&p), g_paged_err) != cudaSuccess) return nullptr;
    return p;
}

static __global__ void paged_error_clear_kernel(int bits) { atomicAnd(&g_paged_err, ~bits); }

int paged_error_clear(int bits) {
    // not a memset: a call on a stream that the default one does not order could set its bit before that
    paged_error_clear_kernel<<<1, 1>>>(bits);
    JYC_LAUNCHED();
    JYC_CUDA(cudaStreamSynchronize(nullptr));
    return JYC_OK;
}

int sm_count() {
    static std::atomic<int> sms[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (dev < 64 && (n = sms[dev].load(std::memory_order_relaxed)) > 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    if (dev < 64) sms[dev].store(n, std::memory_order_relaxed);
    return n;
}

int max_dynamic_smem(const void* kernel, int bytes) {
    // the attribute belongs to the kernel and the device: remembered for the first 64 devices, set again otherwise
    struct Entry {
        const void* kernel;
        uint64_t devices;
    };
    static Entry done[32];
    static std::mutex mu;
    int dev = 0;
    JYC_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lk(mu);
    Entry* e = done;
    while (e < done + 32 && e->kernel && e->kernel != kernel) e++;
    if (e < done + 32 && e->kernel && dev < 64 && (e->devices >> dev & 1)) return JYC_OK;
    JYC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (e < done + 32 && dev < 64) {
        e->kernel = kernel;
        e->devices |= 1ull << dev;
    }
    return JYC_OK;
}

namespace {

__device__ __forceinline__ void paged_flag(int bit) {
    if ((*(volatile int*)&g_paged_err & bit) == 0) atomicOr(&g_paged_err, bit);
}

// Table entry of position `pos` of sequence `seq`, -1 (and the error word)
// when the sequence or the position is out of range; *slot: its place there.
__device__ __forceinline__ int paged_entry(const PagedKV& kv, int seq, int pos, int* slot) {
    const int idx = kv.by_page(pos);
    *slot = pos - idx * kv.p.page_size;
    if (seq < 0 || seq >= kv.num_seqs || idx >= kv.table_stride) {
        paged_flag(kPagedErrPos);
        return -1;
    }
    const int page = __ldg(kv.table + (size_t)seq * kv.table_stride + idx);
    return page == -1 ? INT_MIN : page;  // -1: already flagged
}
// Whether an entry is a page; flags one that is not.
__device__ __forceinline__ bool paged_valid(const PagedKV& kv, int page) {
    if (page >= 0 && page < kv.p.num_pages) return true;
    if (page != -1) paged_flag(kPagedErrPage);
    return false;
}
__device__ __forceinline__ size_t paged_off(const PagedKV& kv, int page, int slot, int h) {
    return (size_t)((long long)page * kv.p.page_stride + (long long)slot * kv.p.pos_stride +
                    (long long)h * kv.p.head_stride);
}
__device__ __forceinline__ size_t paged_soff(const PagedKV& kv, int page, int slot, int h) {
    return (size_t)((long long)page * kv.p.spage_stride + (long long)slot * kv.p.spos_stride +
                    (long long)h * kv.p.shead_stride);
}

__device__ __forceinline__ float4 load4(const float* p, bool vec) {
    if (vec) return __ldg(reinterpret_cast<const float4*>(p));
    return make_float4(__ldg(p), __ldg(p + 1), __ldg(p + 2), __ldg(p + 3));
}

__device__ __forceinline__ float2 load2(const float* p, bool vec) {
    if (vec) return __ldg(reinterpret_cast<const float2*>(p));
    return make_float2(__ldg(p), __ldg(p + 1));
}

// Two pairs rotated by their table entries (rope_pos's rounding: one product
// rounded, one fused sum).
__device__ __forceinline__ float4 rotate4(float4 x, float2 c, float2 s) {
    float4 r;
    r.x = __fmaf_rn(x.x, c.x, -__fmul_rn(x.y, s.x));
    r.y = __fmaf_rn(x.x, s.x, __fmul_rn(x.y, c.x));
    r.z = __fmaf_rn(x.z, c.y, -__fmul_rn(x.w, s.y));
    r.w = __fmaf_rn(x.z, s.y, __fmul_rn(x.w, c.y));
    return r;
}
__device__ __forceinline__ float amax4(float4 x) {
    return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
}
// q8_round of four values without its clamp: |x| <= amax and inv <= 127 / amax
// (1 + 2^-24), so the product stays below 127.5 (and a NaN, or an infinity
// times inv = 0, converts to 0 as there).
__device__ __forceinline__ uint32_t pack4(float4 x, float inv) {
    const int a = __float2int_rn(__fmul_rn(x.x, inv)), b = __float2int_rn(__fmul_rn(x.y, inv));
    const int c = __float2int_rn(__fmul_rn(x.z, inv)), d = __float2int_rn(__fmul_rn(x.w, inv));
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// ---------------------------------------------------------------------------
// Append and read back: append reads 8 hd and writes 2 hd + 8 bytes per row and
// kv head, read the reverse. The bookkeeping of a row is shared: a warp takes
// kRowUnits * (32 / LANES) heads of K or of V of one row. LANES lanes hold a
// head, QUADS groups of four dims each; neighbouring heads lie side by side in a
// warp (whole sectors), and the loads of all units are issued before the first
// is used. They wait for the row's position (a skipped row loads nothing), in
// append not for its page, which only the stores need. (A warp of heads of several rows, each with its own
// position, page and 64-bit offsets, executes 265 instructions per head of 128
// and is bound by them.) Half as many units in flight per warp cost a fifth
// (read of 32768 rows of 8 x 128 88 us against 74), twice as many gain nothing;
// CTAs of 4 warps fill the SMs more evenly than 8 (append 97 -> 91 us).
// Measured at 8 x 128: 16384 rows appended in 55.5 us (floor 26), bound by
// instructions: 168 per head and warp, issue slots 76 % busy with half of the warps
// resident (56 registers). 32768 rows read in 72 us (4.7 TB/s; floor 52): the warps
// wait for position, page and row in a chain (issue slots 55 % busy).
constexpr int kRowUnits = 4, kRowThreads = 128;

struct RowWarp {
    int row, head;  // first head of this lane
    bool is_k;
    int page, slot; // page: as paged_entry returns it, -1: nothing to do
    int pos;
};
template <int LANES>
__device__ __forceinline__ RowWarp row_warp(int rows, int chunks, const FastDiv& by_row, const int* row_seq,
                                            const int* row_pos, const PagedKV& kv, int rope_len) {
    const int w = blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    RowWarp x;
    x.row = by_row(w);
    const int r = w - x.row * 2 * chunks;
    x.is_k = r < chunks;
    x.head = (x.is_k ? r : r - chunks) * kRowUnits * (32 / LANES) + lane / LANES;
    x.page = -1;
    x.pos = -1;
    x.slot = 0;
    if (x.row >= rows) return x;
    x.pos = __ldg(row_pos + x.row);
    const int seq = row_seq ? __ldg(row_seq + x.row) : x.row;
    if (x.pos < 0) return x;
    if (rope_len >= 0 && x.pos >= rope_len) {
        paged_flag(kPagedErrRope);
        return x;
    }
    x.page = paged_entry(kv, seq, x.pos, &x.slot);
    return x;
}

template <int LANES, int QUADS>
__global__ void __launch_bounds__(kRowThreads) paged_append_kernel(const float* K, const float* V, int ld, int rows,
                                                                   int KV, int hd, const int* row_seq,
                                                                   const int* row_pos, PagedKV kv, PagedRope rope,
                                                                   int chunks, FastDiv by_row, bool vec) {
    constexpr int SIDE = 32 / LANES;
    const int sub = threadIdx.x & (LANES - 1), half = hd >> 1, nq = hd >> 2;
    const bool tables = rope.cos_t != nullptr;
    const RowWarp x = row_warp<LANES>(rows, chunks, by_row, row_seq, row_pos, kv, tables ? rope.len : -1);
    if (x.page == -1) return;
    float4 v[kRowUnits][QUADS];
    float2 c[QUADS], sn[QUADS];
    const float* src = (x.is_k ? K : V) + (size_t)x.row * ld + (size_t)x.head * hd;
#pragma unroll
    for (int i = 0; i < kRowUnits; i++)
#pragma unroll
        for (int t = 0; t < QUADS; t++) {
            const int qd = sub + LANES * t;
            v[i][t] = qd < nq && x.head + i * SIDE < KV ? load4(src + i * SIDE * hd + 4 * qd, vec)
                                                        : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    const bool rot = tables && x.is_k;
#pragma unroll
    for (int t = 0; t < QUADS; t++) {
        const int qd = sub + LANES * t;
        const bool use = rot && qd < nq;
        c[t] = use ? load2(rope.cos_t + (size_t)x.pos * half + 2 * qd, vec) : make_float2(1.0f, 1.0f);
        sn[t] = use ? load2(rope.sin_t + (size_t)x.pos * half + 2 * qd, vec) : make_float2(0.0f, 0.0f);
    }
    if (!paged_valid(kv, x.page)) return;
    int8_t* dst = (x.is_k ? kv.p.k : kv.p.v) + paged_off(kv, x.page, x.slot, x.head);
    float* sc = (x.is_k ? kv.p.ks : kv.p.vs) + paged_soff(kv, x.page, x.slot, x.head);
#pragma unroll
    for (int i = 0; i < kRowUnits; i++) {
        float amax = 0.0f;
#pragma unroll
        for (int t = 0; t < QUADS; t++) {
            if (rot) v[i][t] = rotate4(v[i][t], c[t], sn[t]);
            amax = fmaxf(amax, amax4(v[i][t]));
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (x.head + i * SIDE >= KV) continue;
        const float inv = q8_inv(amax);
        if (sub == 0) sc[i * SIDE * kv.p.shead_stride] = q8_scale(amax);
#pragma unroll
        for (int t = 0; t < QUADS; t++) {
            const int qd = sub + LANES * t;
            if (qd < nq)
                *reinterpret_cast<uint32_t*>(dst + i * SIDE * kv.p.head_stride +
                                             4 * (rot ? rope_slot(2 * qd, half) >> 1 : qd)) = pack4(v[i][t], inv);
        }
    }
}

template <int LANES, int QUADS>
__global__ void __launch_bounds__(kRowThreads) paged_read_kernel(float* K, float* V, int ld, int rows, int KV, int hd,
                                                                 const int* row_seq, const int* row_pos, PagedKV kv,
                                                                 int chunks, FastDiv by_row, bool vec) {
    constexpr int SIDE = 32 / LANES;
    const int sub = threadIdx.x & (LANES - 1), nq = hd >> 2;
    const RowWarp x = row_warp<LANES>(rows, chunks, by_row, row_seq, row_pos, kv, -1);
    if (x.page == -1 || !paged_valid(kv, x.page)) return;
    const int8_t* src = (x.is_k ? kv.p.k : kv.p.v) + paged_off(kv, x.page, x.slot, x.head);
    const float* scp = (x.is_k ? kv.p.ks : kv.p.vs) + paged_soff(kv, x.page, x.slot, x.head);
    uint32_t v[kRowUnits][QUADS];
    float sc[kRowUnits];
#pragma unroll
    for (int i = 0; i < kRowUnits; i++) {
        const bool live = x.head + i * SIDE < KV;
        sc[i] = live ? __ldg(scp + i * SIDE * kv.p.shead_stride) : 0.0f;
#pragma unroll
        for (int t = 0; t < QUADS; t++) {
            const int qd = sub + LANES * t;
            v[i][t] = live && qd < nq
                          ? __ldg(reinterpret_cast<const uint32_t*>(src + i * SIDE * kv.p.head_stride) + qd)
                          : 0u;
        }
    }
    float* dst = (x.is_k ? K : V) + (size_t)x.row * ld + (size_t)x.head * hd;
#pragma unroll
    for (int i = 0; i < kRowUnits; i++) {
        if (x.head + i * SIDE >= KV) continue;
#pragma unroll
        for (int t = 0; t < QUADS; t++) {
            const int qd = sub + LANES * t;
            if (qd >= nq) continue;
            float f[4];
            u8x4_to_f32(v[i][t] ^ 0x80808080u, f);
#pragma unroll
            for (int j = 0; j < 4; j++) f[j] = __fmul_rn(f[j], sc[i]);
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
// out = sum_j p_j vs_j v_j / sum_j p_j, p_j = exp(dot_j (ks_j qs) / sqrt(hd)),
// one pass over the keys with a running reference. In base 2, with vs_j =
// 2^e_j f_j (1 <= f_j < 2): b_j = 2^(s_j - ref), w_j = b_j vs_j < 2^(1 + s_j +
// e_j - ref). The reference follows the maximum of s_j + e_j, not of s_j, so
// that the weights neither overflow pairs of fp16 (22 bits) nor lose a small vs
// that carries all the weight; the denominator adds the b_j.
//
// A step reads sum(len) * KV * (2 hd + 8) bytes and is bound by them, so: work
// is a line of units (a unit: TK keys of one kv head of one sequence), cut into
// equal runs for all resident warps whatever the lengths; a warp keeps its next
// units in flight in its own ring in shared memory across the borders of
// sequences and has no barrier in its loop. Heads of 64 or 128 on pages that
// divide a unit or that units divide come by one tensor copy per page, K and V
// each; other shapes by 16- or 4-byte cp.async.
// Keys are the rows of both products and the query heads of a kv head the
// columns: S^T = K Q^T with mma.m16n8k32 s8 (exact dots), then O^T = V^T P^T,
// the weights transposed between them by movmatrix.
//
// The weights go in as fp16 halves hi + lo (22 bits; the largest is held
// within 2^13 .. 2^14, so a lost bit is at most 2^-25, 2^-38 of it) against
// V's bytes as fp16 (exact): mma.m16n8k16, each unit's product from zero and
// added in fp32 with round to nearest (the tensor cores' own sums may
// truncate). 4 heads fill 8 columns with their hi and lo halves: half the
// products (heads of 96: 50 us against 54 with a column a head). Integer
// weights (4 byte columns a head, V unconverted) were as fast at 4 heads and
// slower at 8: 131072 keys of 8 x 128 89 us against 68.
//
// A run that covers an item (a kv head of a sequence) whole writes its rows of
// out; the others leave parts (o, ref, l), which are joined inside the CTA where
// the item ends in it (through shared memory when the CTA has one item only,
// through the workspace otherwise), and by a second kernel where it does not:
// one part per CTA that the item touches.
//
// Measured: 131072 keys of 8 x 128 67 us (floor 43; 7 TB/s while every warp
// streams), 64 sequences of 2048 to 2176 keys of 8 x 64 43 us (floor 23), 45 of
// 1 to 8192 keys of 8 x 128 79 to 85 us by their lengths (floor 60). What is over the floor is the
// ends: finding each warp's run in lens, Q and the page table before the first
// key (8 us), the spread of the warps' ends and the joins (8), the second
// kernel (4).

constexpr float kPaShift = 13.0f;    // the largest weight is in 2^13 .. 2^14
constexpr float kPaLow = -1.7e38f;  // reference before any key: below every score, and its differences stay finite

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// c = v + a b for a constant v, and c += a b
__device__ __forceinline__ void pa_mma_s8(const uint32_t (&a)[4], const uint32_t (&b)[2], int v, int (&c)[4]) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "r"(v));
}
__device__ __forceinline__ void pa_mma_s8(const uint32_t (&a)[4], const uint32_t (&b)[2], int (&c)[4]) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void pa_mma_f16(const uint32_t (&a)[4], const uint32_t (&b)[2], float v, float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(v));
}
__device__ __forceinline__ void pa_mma_f16(const uint32_t (&a)[4], const uint32_t (&b)[2], float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// 8 x 8 halves, lane (g, t) holding (g, 2 t) and (g, 2 t + 1), transposed
__device__ __forceinline__ uint32_t pa_transpose(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void pa_ldsm(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void pa_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// The cache is read once a step: its lines leave L2 first, so that code, queries and parts stay there
// (measured: without the hint a kernel's end runs at DRAM latency, instruction by instruction).
// Scales of neighbouring heads may share a sector, which other SMs want too: no hint.
__device__ __forceinline__ void pa_copy_scale(uint32_t dst, const float* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
template <int N>
__device__ __forceinline__ void pa_copy(uint32_t dst, const void* src, uint64_t policy) {
    if (N == 16)
        asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy)
                     : "memory");
    else
        asm volatile("cp.async.ca.shared.global.L2::cache_hint [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "l"(policy)
                     : "memory");
}
// bytes 0, 2 (ODD: 1, 3) of x = q ^ 0x80 as the halves q: 0x6400 | u is 1024 + u
template <bool ODD>
__device__ __forceinline__ uint32_t pa_half2(uint32_t x) {
    const uint32_t m = __byte_perm(x, 0x64646464u, ODD ? 0x4341 : 0x4240);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&m), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t pa_pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Sizes of one instantiation: HDP is the head size rounded up (the columns
// behind it hold whatever the ring held, finite as integers; they meet zero
// query columns and unread output columns), HEADS the query heads of a unit.
template <int HDP, int HEADS, bool TMA>
struct PaCfg {
    static constexpr int TK = HDP <= 128 ? 32 : 16;        // keys of a unit
    // one CTA per SM. Above 64 dims few warps with more units in flight each and room for every accumulator in
    // registers beat more warps with fewer: 131072 keys of 8 x 128, 4 heads each, take 78 us with 12 warps of 2
    // stages, 66 with 8 of 3; 64 sequences of 2112 keys of 8 x 64 take 43 with 12 warps, 47 with 8
    static constexpr int WARPS = HDP <= 64 ? 12 : 8;
    static constexpr int ST = 3;
    static constexpr int E = HEADS <= 8 ? 1 : 2;           // n8 tiles of heads
    static constexpr int ROWS = HEADS;
    static constexpr int VOFF = TK * HDP, SOFF = 2 * TK * HDP, MOFF = SOFF + 8 * TK;
    // K and V; then ks, vs and the valid mask. A tensor copy's swizzle goes by the address: stages on 1024 bytes,
    // the scales behind all of them
    static constexpr int STAGE = TMA ? SOFF : MOFF + 16;
    static constexpr int PART = ROWS * (HDP + 2);        // floats of a partial: o, then (ref, l) per row
    static constexpr int KOFF = ST * STAGE;              // tensor copies: ks and vs of the stages
    static constexpr int FOFF = KOFF + (TMA ? ST * 8 * TK : 0);  // the current unit's keys, a float4 each
    static constexpr int RING = TMA ? (FOFF + 16 * TK + 1023) / 1024 * 1024 : FOFF + 16 * TK;
    static constexpr int SLACK = TMA ? 1024 : 0;         // to align the first stage
    static constexpr int SMEM = WARPS * RING + SLACK;
    static_assert(PART * 4 <= RING, "a partial fits the ring");
    // byte of 16-byte chunk c of row r: chunks are swapped inside groups of 8 (of 4 where a row is no
    // multiple of 128 bytes) so that the 8 rows of an ldmatrix tile lie in distinct banks
    static __device__ __forceinline__ int at(int r, int c) {
        return r * HDP + 16 * (HDP % 128 == 0 ? c ^ (r & 7) : c ^ ((r >> 1) & 3));
    }
};

// What the kernels share about the line of units.
struct PaMaps {
    CUtensorMap k, v;
};
struct PaPlan {
    int units_row;  // kv heads * query blocks
    int qblocks;    // blocks of ROWS query heads per kv head
    int tk;         // keys of a unit
    bool wide_copy; // 16-byte copies
    bool wide_q;    // 16-byte loads of Q, 8-byte ones of the tables
    int box;        // keys of a tensor copy
};
// The line cut into runs: worker w starts at w * base + min(w, rest).
struct PaLine {
    long long base, rest, workers;
    int per_cta;  // workers of a CTA
    __device__ __forceinline__ long long start(long long w) const {
        w = min(w, workers);
        return w * base + min(w, rest);
    }
    __device__ __forceinline__ int worker(long long u) const {  // whose run holds unit u
        const long long big = rest * (base + 1);
        if (u >> 32) return (int)(u < big ? u / (base + 1) : rest + (u - big) / base);
        return (int)(u < big ? (unsigned)u / (unsigned)(base + 1) : (unsigned)rest + (unsigned)(u - big) / (unsigned)base);
    }
};
// Item that starts in a CTA and ends in a later one.
struct PaTail {
    int ctas;  // CTAs after the first that hold parts of it; 0: no such item
    int slot;  // its first part
    int b, r;
    int per_cta;
};
struct PaWork {
    PaTail* tail;      // [CTAs]
    float* part;       // [workers][2][PART]: an item's later part (0), its first (1)
};

__device__ __forceinline__ int pa_len(const PagedAttn& a, int b) {
    int len = a.lens[b];
    if (len <= 0) return 0;
    const int cap = a.kv.table_stride * a.kv.p.page_size;
    if (len > cap) {
        paged_flag(kPagedErrPos);
        len = cap;
    }
    if (a.rope.cos_t && len > a.rope.len) {
        paged_flag(kPagedErrRope);
        len = 0;
    }
    return len;
}
// Runs of U units: as many workers as there are warps, or units; a few per CTA
// at least, whose parts are joined in shared memory.
constexpr int kPaFewWarps = 4;
__device__ __forceinline__ PaLine pa_line(long long U, int ctas, int warps) {
    PaLine l;
    const long long each = U >> 31 ? warps : ((unsigned)U + ctas - 1) / (unsigned)ctas;
    l.per_cta = (int)min((long long)warps, max((long long)kPaFewWarps, each));
    l.workers = min((long long)ctas * l.per_cta, U);
    l.base = l.rest = 0;
    if (U >> 32) {
        l.base = U / l.workers;
        l.rest = U % l.workers;
    } else if (l.workers) {
        l.base = (unsigned)U / (unsigned)l.workers;
        l.rest = (unsigned)U % (unsigned)l.workers;
    }
    return l;
}

struct PaCursor {
    int b, r, t, nt, len;  // sequence, row of units, unit and units in it, length
};
__device__ __forceinline__ void pa_seek(const PagedAttn& a, int tk, PaCursor& c) {
    c.len = 0;
    while (c.b < a.kv.num_seqs && (c.len = pa_len(a, c.b)) == 0) c.b++;
    c.nt = (c.len + tk - 1) / tk;
}
__device__ __forceinline__ void pa_next(const PagedAttn& a, const PaPlan& pl, PaCursor& c, int step) {
    if ((c.t += step) < c.nt) return;
    c.t = 0;
    if (++c.r < pl.units_row) return;
    c.r = 0;
    c.b++;
    pa_seek(a, pl.tk, c);
}

// A wait that did not end at once: gives up after 2^31 SM cycles (about a
// second) and sets the error word; the warp's run then ends with that unit.
__device__ __noinline__ bool pa_wait_slow(uint64_t* bar, uint32_t parity) {
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity))
        if (clock64() - t0 > (1LL << 31)) {
            paged_flag(kPagedErrWait);
            return false;
        }
    return true;
}
__device__ __forceinline__ bool pa_wait(uint64_t* bar, uint32_t parity) {
    return mbar_try_wait(bar, parity) || pa_wait_slow(bar, parity);
}
// box of a map's tensor [page][slot][kv head][dim] -> shared memory (this CTA's)
__device__ __forceinline__ void pa_tensor_copy(uint32_t dst, const CUtensorMap* map, int h, int slot, int page,
                                               uint64_t* bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::"r"(dst),
        "l"(map), "r"(0), "r"(h), "r"(slot), "r"(page), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}

// One warp's sum of parts for RB query rows: every load of a part is in flight
// at once. Lane i holds dims 4 i .. 4 i + 3 of every 128, and (ref, l) of row i % RB.
template <int HDP, int HEADS, bool TMA>
struct PaSum {
    using G = PaCfg<HDP, HEADS, TMA>;
    static constexpr int RB = HDP <= 128 && HEADS >= 8 ? 8 : 4, NV = (HDP + 127) / 128;
    float4 o[RB][NV];
    float ref, l;
    // parts i = first, first + step, ... < np at work slots slot(i), rows r0 .. r0 + rows - 1
    template <class F>
    __device__ __forceinline__ void add(const float* part, int r0, int rows, int np, int first, int step, F slot) {
        const int lane = threadIdx.x & 31;
        ref = kPaLow;
        l = 0.0f;
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll
            for (int d = 0; d < NV; d++) o[r][d] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int i = first; i < np; i += step) {
            const float* p = part + (size_t)slot(i) * G::PART;
            const float2 rl = *reinterpret_cast<const float2*>(p + G::ROWS * HDP + 2 * (r0 + (lane & (RB - 1))));
            float4 x[RB][NV];
#pragma unroll
            for (int r = 0; r < RB; r++)
#pragma unroll
                for (int d = 0; d < NV; d++)
                    x[r][d] = r < rows && 128 * d + 4 * lane < HDP
                                  ? *reinterpret_cast<const float4*>(p + (r0 + r) * HDP + 128 * d + 4 * lane)
                                  : make_float4(0.f, 0.f, 0.f, 0.f);
            const float nr = fmaxf(ref, rl.x), fa = ex2(ref - nr), fb = ex2(rl.x - nr);
            l = __fmaf_rn(l, fa, rl.y * fb);
            ref = nr;
#pragma unroll
            for (int r = 0; r < RB; r++) {
                const float ga = __shfl_sync(0xffffffffu, fa, r), gb = __shfl_sync(0xffffffffu, fb, r);
#pragma unroll
                for (int d = 0; d < NV; d++) {
                    o[r][d].x = __fmaf_rn(o[r][d].x, ga, x[r][d].x * gb);
                    o[r][d].y = __fmaf_rn(o[r][d].y, ga, x[r][d].y * gb);
                    o[r][d].z = __fmaf_rn(o[r][d].z, ga, x[r][d].z * gb);
                    o[r][d].w = __fmaf_rn(o[r][d].w, ga, x[r][d].w * gb);
                }
            }
        }
    }
    __device__ __forceinline__ void store(float* p, int r0, int rows) const {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll
            for (int d = 0; d < NV; d++)
                if (r < rows && 128 * d + 4 * lane < HDP)
                    *reinterpret_cast<float4*>(p + (r0 + r) * HDP + 128 * d + 4 * lane) = o[r][d];
        if (lane < rows) *reinterpret_cast<float2*>(p + G::ROWS * HDP + 2 * (r0 + lane)) = make_float2(ref, l);
    }
    __device__ __forceinline__ void finish(float* out, int rows, int hd) const {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int r = 0; r < RB; r++) {
            const float lr = __shfl_sync(0xffffffffu, l, r), inv = lr == 0.0f ? 0.0f : __fdiv_rn(1.0f, lr);
#pragma unroll
            for (int d = 0; d < NV; d++) {
                const int e = 128 * d + 4 * lane;
                if (r >= rows || e >= hd) continue;
                float* to = out + (size_t)r * hd + e;
                to[0] = o[r][d].x * inv;
                to[1] = o[r][d].y * inv;
                to[2] = o[r][d].z * inv;
                to[3] = o[r][d].w * inv;
            }
        }
    }
};

template <int HDP, int HEADS, bool TMA>
__global__ void __launch_bounds__(PaCfg<HDP, HEADS, TMA>::WARPS * 32, 1)
    paged_attention_kernel(PagedAttn a, PaPlan pl, PaWork work, const __grid_constant__ PaMaps maps) {
    using G = PaCfg<HDP, HEADS, TMA>;
    constexpr int TK = G::TK, ST = G::ST, WARPS = G::WARPS, ROWS = G::ROWS, E = G::E;
    constexpr int NK = HDP / 32, NM = TK / 16, ND = HDP / 16;
    extern __shared__ __align__(128) unsigned char pa_raw[];
    unsigned char* const pa_sm = TMA ? pa_raw + (-smem_u32(pa_raw) & 1023u) : pa_raw;
    __shared__ __align__(8) uint64_t s_bar[WARPS][ST][2];  // K, V
    __shared__ long long s_scan[WARPS], s_ex[WARPS * 32];
    const uint64_t policy = policy_evict_first();
    __shared__ PaCursor s_cur[WARPS];
    __shared__ long long s_first[WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int B = a.kv.num_seqs, group = a.H / a.KV, hd = TMA ? HDP : a.hd;
    griddep_launch();
    if (TMA && lane == 0) {
        if (warp == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.k) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.v) : "memory");
        }
        for (int i = 0; i < 2 * ST; i++) mbar_init(&s_bar[warp][0][i], 1);
        mbar_fence_init();
    }

    // where the units of each sequence lie in the line
    const int per = (B + WARPS * 32 - 1) / (WARPS * 32);
    const int bs = min(B, tid * per), be = min(B, bs + per);
    long long mine = 0;
    bool none = false;  // one of this CTA's share of sequences has no key
    for (int b = bs; b < be; b++) {
        const int len = pa_len(a, b);
        mine += (len + TK - 1) / TK;
        none |= len == 0 && b % gridDim.x == blockIdx.x;
    }
    mine *= pl.units_row;
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    if (lane == 31) s_scan[warp] = incl;
    if (__syncthreads_or(none))  // rows of zeros
        for (int b = blockIdx.x; b < B; b += gridDim.x)
            if (pa_len(a, b) == 0)
                for (int e = tid; e < a.H * hd; e += WARPS * 32) a.out[(size_t)b * a.ldo + e] = 0.0f;
    long long U = 0, ex = incl - mine;
    for (int w = 0; w < WARPS; w++) {
        if (w < warp) ex += s_scan[w];
        U += s_scan[w];
    }
    const PaLine line = pa_line(U, gridDim.x, WARPS);
    const long long w0 = (long long)blockIdx.x * line.per_cta;
    s_ex[tid] = ex;
    __syncthreads();
    {
        // warp: where its run starts (the last thread's segment that starts at or before it)
        const long long u = line.start(w0 + warp);
        if (warp < line.per_cta && u < U) {
            int lo = 0;
#pragma unroll
            for (int i = 1 << (31 - __builtin_clz(WARPS * 32)); i > 0; i >>= 1)
                if (lo + i < WARPS * 32 && s_ex[lo + i] <= u) lo += i;
            long long at = s_ex[lo];
            for (int b = min(B, lo * per); b < B; b++) {
                const int len = pa_len(a, b), nt = (len + TK - 1) / TK;
                const long long n = (long long)nt * pl.units_row;
                if (u < at + n) {
                    const long long k = u - at;
                    const int r = k >> 31 ? (int)(k / nt) : (int)k / nt, t0 = (int)(k - (long long)r * nt);
                    s_cur[warp] = PaCursor{b, r, t0, nt, len};
                    s_first[warp] = u - t0;  // first unit of the item that the run starts in
                    break;
                }
                at += n;
            }
        }
    }
    __syncthreads();

    const bool worker = warp < line.per_cta;
    const long long u0 = line.start(w0 + warp), c0 = line.start(w0), c1 = line.start(w0 + line.per_cta);
    // every run of the CTA inside one item: its warps take units in turn (neighbours in memory at the same time)
    // and are joined below. whole: and they are all of it
    bool joint = false, whole = false;
    if (c1 > c0) {
        const long long first = s_first[0], end = first + s_cur[0].nt;
        joint = c1 <= end;
        whole = c0 == first && c1 == end;
    }
    int count = worker ? (int)(line.start(w0 + warp + 1) - u0) : 0;
    const int step = joint ? line.per_cta : 1;
    unsigned char* ring = pa_sm + warp * G::RING;
    const uint32_t ring_a = smem_u32(ring);
    PaCursor cur = PaCursor{0, 0, 0, 0, 0};
    long long item0 = 0;
    if (joint) {
        cur = s_cur[0];
        cur.t += warp;
        const int units = (int)(c1 - c0);
        count = worker && warp < units ? (units - warp + step - 1) / step : 0;
    } else if (count > 0) {
        cur = s_cur[warp];
        item0 = s_first[warp];
    }
    const bool alone = whole && c1 - c0 == 1;
    if (tid == 0) work.tail[blockIdx.x].ctas = 0;

    // copies: lane j looks up the page of key j of a unit one step before the unit's copies are issued
    PaCursor nx = cur;
    int issued = 0;  // units whose pages are looked up
    int pg = -1, slot = 0, h = -1;
    long long hoff = 0, hsoff = 0;  // of kv head h
    bool ok = false;
    auto lookup = [&] {
        ok = false;
        if (issued < count) {
            const int pos = nx.t * TK + lane, hn = pl.qblocks == 1 ? nx.r : nx.r / pl.qblocks;
            if (hn != h) {
                h = hn;
                hoff = (long long)h * a.kv.p.head_stride;
                hsoff = (long long)h * a.kv.p.shead_stride;
            }
            if (lane < TK && pos < nx.len) {
                const int idx = a.kv.by_page(pos);
                slot = pos - idx * a.kv.p.page_size;
                pg = __ldg(a.kv.table + (size_t)nx.b * a.kv.table_stride + idx);
                ok = true;
            }
            pa_next(a, pl, nx, step);
        }
        issued++;
    };
    bool lead = false;
    unsigned bytes = 0u, counts = 0u;  // counts: whether this lane's key counts, of the unit issued last in bit 0
    constexpr int LPR = HDP <= 64 ? 4 : HDP <= 128 ? 8 : 16, RPI = 32 / LPR;  // lanes per row, rows per step
    const int cc = (lane & (LPR - 1)) * 16, cr = lane / LPR;
    const int8_t* const kcol = a.kv.p.k + cc;
    const int8_t* const vcol = a.kv.p.v + cc;
    // tensor copies of the unit that was looked up last: K and its keys' scales (lane j copies and reads key j's),
    // then V
    auto issue_k = [&](int st) {
        if (ok && (unsigned)pg >= (unsigned)a.kv.p.num_pages) {
            paged_flag(kPagedErrPage);
            ok = false;
        }
        counts = counts << 1 | (ok ? 1u : 0u);
        lead = ok && (lane & (pl.box - 1)) == 0;
        bytes = __popc(__ballot_sync(0xffffffffu, lead)) * pl.box * HDP;
        uint64_t* bar = &s_bar[warp][st][0];
        if (lane == 0) mbar_expect_tx(bar, bytes);
        __syncwarp();
        if (lead) pa_tensor_copy(ring_a + st * G::STAGE + lane * HDP, &maps.k, h, slot, pg, bar, policy);
        if (ok) {
            const long long so = (long long)pg * a.kv.p.spage_stride + (long long)slot * a.kv.p.spos_stride + hsoff;
            pa_copy_scale(ring_a + G::KOFF + st * 8 * TK + 4 * lane, a.kv.p.ks + so);
            pa_copy_scale(ring_a + G::KOFF + st * 8 * TK + 4 * TK + 4 * lane, a.kv.p.vs + so);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto issue_v = [&](int st) {
        uint64_t* bar = &s_bar[warp][st][1];
        if (lane == 0) mbar_expect_tx(bar, bytes);
        __syncwarp();
        if (lead) pa_tensor_copy(ring_a + st * G::STAGE + G::VOFF + lane * HDP, &maps.v, h, slot, pg, bar, policy);
    };
    auto issue = [&](int st) {  // K, V and scales by cp.async
        if (ok && (unsigned)pg >= (unsigned)a.kv.p.num_pages) {
            paged_flag(kPagedErrPage);
            ok = false;
        }
        const uint32_t base = ring_a + st * G::STAGE;
        const unsigned mask = __ballot_sync(0xffffffffu, ok);
        long long off = 0;
        if (ok) {
            off = (long long)pg * a.kv.p.page_stride + (long long)slot * a.kv.p.pos_stride + hoff;
            const long long so = (long long)pg * a.kv.p.spage_stride + (long long)slot * a.kv.p.spos_stride + hsoff;
            pa_copy_scale(base + G::SOFF + 4 * lane, a.kv.p.ks + so);
            pa_copy_scale(base + G::SOFF + 4 * TK + 4 * lane, a.kv.p.vs + so);
        }
        if (lane == 0) *reinterpret_cast<unsigned*>(ring + st * G::STAGE + G::MOFF) = mask;
        if (pl.wide_copy) {
            const bool all = mask == (TK == 32 ? ~0u : (1u << (TK & 31)) - 1u);
#pragma unroll
            for (int i = 0; i < TK / RPI; i++) {
                const int row = i * RPI + cr;
                const long long o = __shfl_sync(0xffffffffu, off, row);
                if (cc < hd && (all || ((mask >> row) & 1))) {
                    const uint32_t dst = base + G::at(row, cc / 16);
                    pa_copy<16>(dst, kcol + o, policy);
                    pa_copy<16>(dst + G::VOFF, vcol + o, policy);
                }
            }
        } else {
            for (int row = 0; row < TK; row++) {
                const long long o = __shfl_sync(0xffffffffu, off, row);
                if (!((mask >> row) & 1)) continue;
                for (int c = lane; c * 4 < hd; c += 32) {
                    const uint32_t dst = base + G::at(row, c / 4) + (c & 3) * 4;
                    pa_copy<4>(dst, a.kv.p.k + o + c * 4, policy);
                    pa_copy<4>(dst + G::VOFF, a.kv.p.v + o + c * 4, policy);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto begin = [&] {  // copies of the first units
#pragma unroll 1
        for (int i = 0; i < (TMA ? ST : ST - 1); i++) {
            if constexpr (TMA) {
                issue_k(i);
                issue_v(i);
            } else {
                issue(i);
            }
            lookup();
        }
    };

    // lane (g, t): query head g (and g + 8) as B fragments, bytes 4 t .. 4 t + 3 of every 16; of the results the
    // heads 2 t, 2 t + 1 (and 8 more), for which it keeps the reference, its share of the sum, and the dims 2 g,
    // 2 g + 1 of every 16
    uint32_t qf[NK][E][2];
    float qsl[E][2], ref[E][2], l[E][2], o[ND][E][4];
    bool fresh = true, tail = false;  // tail: the run ends inside an item that it starts
    bool gave_up = false;
    int st = 0;
    uint32_t phase = 0u;
    const float up = __fmul_rn(a.scale, 1.44269504088896341f);

    for (int n = 0; n < count; n++) {
        if (fresh) {
            // the item's query heads: rotated and quantised per head
            fresh = false;
            if (n == 0) lookup();
            const int qb = cur.r % pl.qblocks, kvh = cur.r / pl.qblocks;
            const int half = hd >> 1;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int row = qb * ROWS + 8 * e + (HEADS <= 4 ? g & 3 : g);
                const bool live = row < group;
                const float* q = a.Q + (size_t)cur.b * a.ldq + (size_t)(kvh * group + (live ? row : 0)) * hd;
                const size_t tp = (size_t)(cur.len - 1) * half;
                const bool rot = a.rope.cos_t != nullptr;
                float4 x[2 * NK];
                float2 c[2 * NK], sn[2 * NK];
                float amax = 0.0f;
#pragma unroll
                for (int i = 0; i < 2 * NK; i++) {
                    int src = 4 * i + t;  // quad stored in slot 4 i + t
                    x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (!live || 4 * src >= hd) continue;
                    if (rot) {
                        src = rope_slot(2 * src, half) >> 1;  // its own inverse
                        c[i] = load2(a.rope.cos_t + tp + 2 * src, pl.wide_q);
                        sn[i] = load2(a.rope.sin_t + tp + 2 * src, pl.wide_q);
                    }
                    x[i] = load4(q + 4 * src, pl.wide_q);
                }
                // the queries are on their way before the first copies fill the memory system's queues
                if (e == 0 && n == 0) begin();
#pragma unroll
                for (int i = 0; i < 2 * NK; i++) {
                    if (rot && live && 4 * (4 * i + t) < hd) x[i] = rotate4(x[i], c[i], sn[i]);
                    amax = fmaxf(amax, amax4(x[i]));
                }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                const float inv = q8_inv(amax), sc = __fmul_rn(q8_scale(amax), up);
#pragma unroll
                for (int i = 0; i < 2 * NK; i++) qf[i >> 1][e][i & 1] = pack4(x[i], inv);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    qsl[e][i] = __shfl_sync(0xffffffffu, sc, 4 * (2 * t + i));
                    ref[e][i] = kPaLow;
                    l[e][i] = 0.0f;
                }
#pragma unroll
                for (int d = 0; d < ND; d++) o[d][e][0] = o[d][e][1] = o[d][e][2] = o[d][e][3] = 0.0f;
            }
        }
        bool in = false;
        float kscale, vscale;
        if constexpr (TMA) {
            in = (counts >> (ST - 1)) & 1u;
            asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
            const float* sc = reinterpret_cast<const float*>(ring + G::KOFF + st * 8 * TK);
            kscale = sc[lane];
            vscale = in ? sc[TK + lane] : 0.0f;
            if (!pa_wait(&s_bar[warp][st][0], phase)) gave_up = true;
        } else {
            // the next unit's copies go to the stage that the last iteration read
            __syncwarp();
            issue(st == 0 ? ST - 1 : st - 1);
            lookup();
            asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
            __syncwarp();
        }
        const unsigned char* sb = ring + st * G::STAGE;
        const uint32_t base = ring_a + st * G::STAGE;
        // lane j: key j's {ks, 0 or -inf, e, vs}; a key that does not count has a score of -inf and vs = 0.
        // e is kept within 2^-64..2^126: the quantiser's scales are 0 or above 2^-34
        float4* keys = reinterpret_cast<float4*>(ring + G::FOFF);
        if (lane < TK) {
            if constexpr (!TMA) {
                in = (*reinterpret_cast<const unsigned*>(sb + G::MOFF) >> lane) & 1;
                const float* sc = reinterpret_cast<const float*>(sb + G::SOFF);
                kscale = sc[lane];
                vscale = in ? sc[TK + lane] : 0.0f;
            }
            const int ex = min(max((int)((__float_as_uint(vscale) >> 23) & 255u), 63), 253) - 127;
            // 0, or NaN where ks or vs is not a number or infinite: so is the row then, whatever its weight
            const float bias = __fsub_rn(kscale, kscale) + __fsub_rn(vscale, vscale);
            keys[lane] = in ? make_float4(kscale, bias, (float)ex, vscale) : make_float4(0.0f, -INFINITY, 0.0f, 0.0f);
        }
        __syncwarp();

        // scores of keys 16 m + g, + 8 and heads 2 t, + 1, in base 2; the dots start at the bits of
        // 1.5 * 2^23 (|dot| <= 256 * 127^2 < 2^22), so an exact subtraction makes them floats
        float s[NM][E][4], vs[NM][2];
        float top[E][2];
#pragma unroll
        for (int e = 0; e < E; e++) top[e][0] = top[e][1] = -INFINITY;
#pragma unroll
        for (int m = 0; m < NM; m++) {
            int c[E][4];
#pragma unroll
            for (int k = 0; k < NK; k++) {
                uint32_t kf[4];
                pa_ldsm(base + G::at(16 * m + (lane & 15), 2 * k + (lane >> 4)), kf);
#pragma unroll
                for (int e = 0; e < E; e++) {
                    if (k == 0)
                        pa_mma_s8(kf, qf[k][e], 0x4B400000, c[e]);
                    else
                        pa_mma_s8(kf, qf[k][e], c[e]);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float4 key = keys[16 * m + 8 * i + g];
                vs[m][i] = key.w;
#pragma unroll
                for (int e = 0; e < E; e++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const float dot = __fsub_rn(__int_as_float(c[e][2 * i + j]), 12582912.0f);
                        const float v = __fmaf_rn(dot, __fmul_rn(key.x, qsl[e][j]), key.y);
                        s[m][e][2 * i + j] = v;
                        top[e][j] = fmaxf(top[e][j], v + key.z);
                    }
            }
        }
        if constexpr (TMA) {  // K is read: the unit ST ahead may take its place
            if (!__any_sync(0xffffffffu, gave_up)) issue_k(st);
        }
        float al[E][2];
#pragma unroll
        for (int e = 0; e < E; e++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                float x = top[e][j];
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                x = fmaxf(ref[e][j], x - kPaShift);
                al[e][j] = ex2(ref[e][j] - x);
                ref[e][j] = x;
                l[e][j] *= al[e][j];
            }
        // weights, transposed into B fragments: column g, keys 16 m + 2 t, + 1 and 8 later. A column is a head;
        // of 4 heads or fewer, columns 0-3 are the hi halves and 4-7 the lo halves of the same heads
        uint32_t hi[NM][E][2], lo[NM][E][2];
#pragma unroll
        for (int m = 0; m < NM; m++)
#pragma unroll
            for (int e = 0; e < E; e++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float b0 = ex2(s[m][e][2 * i] - ref[e][0]), b1 = ex2(s[m][e][2 * i + 1] - ref[e][1]);
                    l[e][0] += b0;
                    l[e][1] += b1;
                    const float w0 = b0 * vs[m][i], w1 = b1 * vs[m][i];
                    const uint32_t ph = pa_pack(w0, w1);
                    const float2 hf = __half22float2(*reinterpret_cast<const __half2*>(&ph));
                    const uint32_t pl2 = pa_pack(w0 - hf.x, w1 - hf.y);
                    hi[m][e][i] = pa_transpose(HEADS <= 4 && t >= 2 ? pl2 : ph);
                    if (HEADS > 4) lo[m][e][i] = pa_transpose(pl2);
                }
        if constexpr (TMA)
            if (!pa_wait(&s_bar[warp][st][1], phase)) gave_up = true;
        // P.V: a transposed load gives lane (g, t) dims 2 g, 2 g + 1 of keys 2 t, 2 t + 1: the even dims are
        // rows g of the tile, the odd ones rows g + 8
#pragma unroll
        for (int d = 0; d < ND; d += 2) {
            float c[2][E][4];
#pragma unroll
            for (int m = 0; m < NM; m++) {
                uint32_t v[4];
                pa_ldsm_t(base + G::VOFF + G::at(16 * m + (lane & 15), d + (lane >> 4)), v);
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] ^= 0x80808080u;
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const uint32_t vf[4] = {pa_half2<false>(v[2 * i]), pa_half2<true>(v[2 * i]),
                                            pa_half2<false>(v[2 * i + 1]), pa_half2<true>(v[2 * i + 1])};
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        if (m == 0)
                            pa_mma_f16(vf, hi[m][e], 0.0f, c[i][e]);
                        else
                            pa_mma_f16(vf, hi[m][e], c[i][e]);
                        if (HEADS > 4) pa_mma_f16(vf, lo[m][e], c[i][e]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int e = 0; e < E; e++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        o[d + i][e][j] = __fmaf_rn(o[d + i][e][j], al[e][j & 1], c[i][e][j]);
        }
        if constexpr (TMA) {
            if (__any_sync(0xffffffffu, gave_up)) {
                count = n + 1;  // the run ends here
                gave_up = true;
            } else {
                issue_v(st);
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
        // the end of an item or of the run
        if (HEADS <= 4)  // lanes t and t + 2 hold the sums of hi and lo halves of the same heads
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int j = 0; j < 4; j++) o[d][0][j] += __shfl_xor_sync(0xffffffffu, o[d][0][j], 2);
#pragma unroll
        for (int e = 0; e < E; e++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[e][j] += __shfl_xor_sync(0xffffffffu, l[e][j], x);
        const bool from_start = item0 >= u0;
        if (joint ? alone : from_start && item_end) {
            const int qb = cur.r % pl.qblocks, kvh = cur.r / pl.qblocks;
#pragma unroll
            for (int e = 0; e < E; e++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int row = qb * ROWS + 8 * e + 2 * t + j;
                    if (row >= group) continue;
                    float* out = a.out + (size_t)cur.b * a.ldo + (size_t)(kvh * group + row) * hd;
                    const float inv = l[e][j] == 0.0f ? 0.0f : __fdiv_rn(1.0f, l[e][j]);
#pragma unroll
                    for (int d = 0; d < ND; d++)
                        if (16 * d + 2 * g < hd) {
                            out[16 * d + 2 * g] = o[d][e][j] * inv;
                            out[16 * d + 2 * g + 1] = o[d][e][2 + j] * inv;
                        }
                }
        } else {
            if (joint) break;  // o, ref and l stay in registers
            tail = from_start;
            float* part = work.part + ((size_t)(w0 + warp) * 2 + (from_start ? 1 : 0)) * G::PART;
#pragma unroll
            for (int e = 0; e < E; e++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int row = 8 * e + 2 * t + j;
                    if (row >= ROWS) continue;
#pragma unroll
                    for (int d = 0; d < ND; d++)
                        *reinterpret_cast<float2*>(part + row * HDP + 16 * d + 2 * g) =
                            make_float2(o[d][e][j], o[d][e][2 + j]);
                    if (g == 0)
                        *reinterpret_cast<float2*>(part + ROWS * HDP + 2 * row) = make_float2(ref[e][j], l[e][j]);
                }
        }
        if (n + 1 < count) {
            item0 += cur.nt;
            pa_next(a, pl, cur, 1);
            fresh = true;
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (TMA && gave_up)  // the copies that are still on their way write to this CTA's memory
        for (int i = 0; i < ST; i++) {
            pa_wait(&s_bar[warp][st][0], phase);
            pa_wait(&s_bar[warp][st][1], phase);
            if (++st == ST) {
                st = 0;
                phase ^= 1u;
            }
        }
    // CTAs behind this one that hold parts of an item that ends at unit `end`
    auto later = [&](long long end) { return (int)(line.worker(end - 1) / line.per_cta) - (int)blockIdx.x; };
    if (!joint) {
        // the items that this CTA's runs share: the warp where one starts joins its parts (warp 0 those of the
        // item that came into the CTA), in place
        __syncthreads();
        if (c1 == c0) return;
        const long long first = s_first[0], end0 = first + s_cur[0].nt;
        for (int pass = warp == 0 ? 0 : 1; pass < 2; pass++) {
            const bool head = pass == 0;
            if (head ? first >= c0 : !tail) continue;
            const long long end = head ? end0 : item0 + cur.nt;
            const int own = (int)(w0 + warp) * 2 + (head ? 0 : 1);
            int np = 1;
            while (warp + np < line.per_cta && line.start(w0 + warp + np) < end) np++;
            const PaCursor it = head ? s_cur[0] : cur;
            const bool ends = !head && end <= c1;
            if (!head && !ends && lane == 0)
                work.tail[blockIdx.x] = PaTail{later(end), own, it.b, it.r, line.per_cta};
            if (np == 1) continue;
            const int qb = it.r % pl.qblocks, kvh = it.r / pl.qblocks;
            auto slot_of = [&](int i) { return i == 0 ? own : (int)(w0 + warp + i) * 2; };
            for (int r0 = 0; r0 < ROWS && qb * ROWS + r0 < group; r0 += PaSum<HDP, HEADS, TMA>::RB) {
                PaSum<HDP, HEADS, TMA> sum;
                const int rows = min(PaSum<HDP, HEADS, TMA>::RB, group - qb * ROWS - r0);
                sum.add(work.part, r0, rows, np, 0, 1, slot_of);
                if (ends)
                    sum.finish(a.out + (size_t)it.b * a.ldo + (size_t)(kvh * group + qb * ROWS + r0) * hd, rows, hd);
                else
                    sum.store(work.part + (size_t)own * G::PART, r0, rows);
            }
        }
        return;
    }
    if (alone) return;  // written

    // join the CTA's workers (their rings are free now)
    float* buf = reinterpret_cast<float*>(ring);
    if (worker)
#pragma unroll
        for (int e = 0; e < E; e++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int row = 8 * e + 2 * t + j;
                if (row >= ROWS) continue;
                if (count > 0)
#pragma unroll
                    for (int d = 0; d < ND; d++)
                        *reinterpret_cast<float2*>(buf + row * HDP + 16 * d + 2 * g) =
                            make_float2(o[d][e][j], o[d][e][2 + j]);
                if (g == 0)
                    *reinterpret_cast<float2*>(buf + ROWS * HDP + 2 * row) =
                        count > 0 ? make_float2(ref[e][j], l[e][j]) : make_float2(kPaLow, 0.0f);
            }
    __syncthreads();
    const PaCursor c = s_cur[0];
    const int qb = c.r % pl.qblocks, kvh = c.r / pl.qblocks;
    const int own = (int)w0 * 2 + (c0 == s_first[0] ? 1 : 0);
    float* part = work.part + (size_t)own * G::PART;
    if (tid == 0 && !whole && c0 == s_first[0])
        work.tail[blockIdx.x] = PaTail{later(s_first[0] + c.nt), own, c.b, c.r, line.per_cta};
    for (int i = tid; i < ROWS * HDP / 4; i += WARPS * 32) {
        const int row = i / (HDP / 4), d = i % (HDP / 4) * 4;
        float M = kPaLow, L = 0.0f;
        float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int w = 0; w < line.per_cta; w++)
            M = fmaxf(M, reinterpret_cast<const float*>(pa_sm + w * G::RING)[ROWS * HDP + 2 * row]);
#pragma unroll 1
        for (int w = 0; w < line.per_cta; w++) {
            const float* wb = reinterpret_cast<const float*>(pa_sm + w * G::RING);
            const float wr = wb[ROWS * HDP + 2 * row], wl = wb[ROWS * HDP + 2 * row + 1];
            if (wl == 0.0f) continue;  // no key (a warp without units left no o)
            const float f = ex2(wr - M);
            const float4 x = *reinterpret_cast<const float4*>(wb + row * HDP + d);
            L = __fmaf_rn(f, wl, L);
            O = make_float4(__fmaf_rn(f, x.x, O.x), __fmaf_rn(f, x.y, O.y), __fmaf_rn(f, x.z, O.z), __fmaf_rn(f, x.w, O.w));
        }
        if (whole) {
            if (qb * ROWS + row < group && d < hd) {
                float* out = a.out + (size_t)c.b * a.ldo + (size_t)(kvh * group + qb * ROWS + row) * hd + d;
                const float inv = L == 0.0f ? 0.0f : __fdiv_rn(1.0f, L);
                out[0] = O.x * inv;
                out[1] = O.y * inv;
                out[2] = O.z * inv;
                out[3] = O.w * inv;
            }
        } else {
            *reinterpret_cast<float4*>(part + row * HDP + d) = O;
            if (d == 0) *reinterpret_cast<float2*>(part + ROWS * HDP + 2 * row) = make_float2(M, L);
        }
    }
}

// The items that start in one CTA of the kernel above and end in a later one:
// a CTA each. Warp w adds parts w, w + 8, ..., then the warps' sums are joined
// in shared memory.
constexpr int kPaJoinWarps = 8;
template <int HDP, int HEADS, bool TMA>
__global__ void __launch_bounds__(kPaJoinWarps * 32) paged_join_kernel(PagedAttn a, PaPlan pl, PaWork work) {
    using G = PaCfg<HDP, HEADS, TMA>;
    using Sum = PaSum<HDP, HEADS, TMA>;
    constexpr int ROWS = G::ROWS, NV = Sum::NV, RB = Sum::RB;
    __shared__ __align__(16) float s_o[kPaJoinWarps][RB][HDP];
    __shared__ float2 s_rl[kPaJoinWarps][RB];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = a.H / a.KV, hd = a.hd;
    griddep_wait();
    const PaTail tail = work.tail[blockIdx.x];
    if (tail.ctas == 0) return;
    const int np = tail.ctas + 1, qb = tail.r % pl.qblocks, kvh = tail.r / pl.qblocks;
    auto slot_of = [&](int i) { return i == 0 ? tail.slot : ((int)blockIdx.x + i) * tail.per_cta * 2; };
    for (int r0 = 0; r0 < ROWS && qb * ROWS + r0 < group; r0 += RB) {
        const int rows = min(RB, group - qb * ROWS - r0);
        Sum sum;
        sum.add(work.part, r0, rows, np, warp, kPaJoinWarps, slot_of);
        if (r0) __syncthreads();  // the last row block's sums are read
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll
            for (int d = 0; d < NV; d++)
                if (128 * d + 4 * lane < HDP) *reinterpret_cast<float4*>(&s_o[warp][r][128 * d + 4 * lane]) = sum.o[r][d];
        if (lane < RB) s_rl[warp][lane] = make_float2(sum.ref, sum.l);
        __syncthreads();
        const int used = min(np, kPaJoinWarps);
        for (int i = tid; i < rows * HDP; i += kPaJoinWarps * 32) {
            const int r = i / HDP, d = i % HDP;
            float M = kPaLow, L = 0.0f, O = 0.0f;
            for (int w = 0; w < used; w++) M = fmaxf(M, s_rl[w][r].x);
            for (int w = 0; w < used; w++) {
                const float f = ex2(s_rl[w][r].x - M);
                L = __fmaf_rn(f, s_rl[w][r].y, L);
                O = __fmaf_rn(f, s_o[w][r][d], O);
            }
            if (d < hd)
                a.out[(size_t)tail.b * a.ldo + (size_t)(kvh * group + qb * ROWS + r0 + r) * hd + d] =
                    L == 0.0f ? 0.0f : __fdiv_rn(O, L);
        }
    }
}

// The cache of rows r0, r0 + 1, ... when a row is its own sequence.
PagedKV shifted(PagedKV kv, const int* row_seq, int r0) {
    if (!row_seq) {
        kv.table += (size_t)r0 * kv.table_stride;
        kv.num_seqs -= r0;
    }
    return kv;
}

size_t align16(size_t n) { return (n + 15) / 16 * 16; }

template <int HDP, int HEADS, bool TMA>
size_t pa_work_bytes(int ctas, unsigned char* base, PaWork* w) {
    const size_t workers = (size_t)ctas * PaCfg<HDP, HEADS, TMA>::WARPS;
    const size_t at = align16(ctas * sizeof(PaTail));
    if (w) *w = PaWork{reinterpret_cast<PaTail*>(base), reinterpret_cast<float*>(base + at)};
    return at + workers * 2 * PaCfg<HDP, HEADS, TMA>::PART * sizeof(float);
}

// Map of a cache array as [page][slot][kv head][dim], boxes of `box` slots of one head.
int pa_map(CUtensorMap* m, int8_t* base, const PagedAttn& a, int box) {
    static std::atomic<void*> entry;
    void* fn = entry.load(std::memory_order_acquire);
    if (!fn) {
        cudaDriverEntryPointQueryResult found;
        JYC_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found));
        if (found != cudaDriverEntryPointSuccess || !fn) return cuda_fail(cudaErrorNotSupported, "cuTensorMapEncodeTiled");
        entry.store(fn, std::memory_order_release);
    }
    const jyc_kv_pages& p = a.kv.p;
    const cuuint64_t dims[4] = {(cuuint64_t)a.hd, (cuuint64_t)a.KV, (cuuint64_t)p.page_size, (cuuint64_t)p.num_pages};
    // the stride of a dimension of one entry is not used, but has to be one
    const cuuint64_t strides[3] = {(cuuint64_t)(a.KV > 1 ? p.head_stride : a.hd),
                                   (cuuint64_t)(p.page_size > 1 ? p.pos_stride : a.hd),
                                   (cuuint64_t)(p.num_pages > 1 ? p.page_stride : a.hd)};
    const cuuint32_t boxes[4] = {(cuuint32_t)a.hd, 1, (cuuint32_t)box, 1}, step[4] = {1, 1, 1, 1};
    // L2 promotion to 64 bytes: a row is all that a place of a page may hold of its head (heads of 64, 64 sequences of
    // 2112 keys: 44 us, 47 with 128 bytes, 60 with 256)
    const CUresult r = reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(fn)(
        m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, base, dims, strides, boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
        a.hd == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_64B,
        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return cuda_fail(cudaErrorInvalidValue, "cuTensorMapEncodeTiled");
    return JYC_OK;
}

// Tensor copies need rows of 64 or 128 bytes, strides below 2^40 that are multiples of 16 bytes, pages that
// a unit of 32 keys fills or that fill a unit, and boxes that start on 128 bytes of shared memory. Against 16-byte
// cp.async: 64 sequences of 2112 keys of 8 x 64 44 us to 61, 45 of 1 to 8192 keys of 8 x 128 85 to 88, but one of
// 131072 keys 67 to 62.
bool pa_tensor_copies(const PagedAttn& a, bool aligned) {
    const jyc_kv_pages& p = a.kv.p;
    const long long far = std::max(p.page_stride, std::max(p.pos_stride, p.head_stride));
    const bool nonzero = (p.head_stride > 0 || a.KV == 1) && (p.pos_stride > 0 || p.page_size == 1) &&
                         (p.page_stride > 0 || p.num_pages == 1);
    return aligned && nonzero && far < (1LL << 40) && (a.hd == 64 || a.hd == 128) &&
           (p.page_size % 32 == 0 || (32 % p.page_size == 0 && p.page_size * a.hd % 128 == 0));
}

template <int HDP, int HEADS, bool TMA>
int pa_launch(const PagedAttn& a, PaPlan pl, int sms, void* work, cudaStream_t s) {
    using G = PaCfg<HDP, HEADS, TMA>;
    if (int e = max_dynamic_smem(reinterpret_cast<const void*>(paged_attention_kernel<HDP, HEADS, TMA>), G::SMEM))
        return e;
    const long long cap = (long long)a.kv.table_stride * a.kv.p.page_size, tiles = (cap + G::TK - 1) / G::TK;
    const long long items = (long long)a.kv.num_seqs * pl.units_row;
    // no more CTAs than the longest possible lengths have units for
    const long long units = tiles >= (1LL << 31) / items ? 1LL << 31 : items * tiles;
    const int ctas = (int)std::max(1LL, std::min((long long)sms, (units + kPaFewWarps - 1) / kPaFewWarps));
    pl.tk = G::TK;
    PaMaps maps{};
    if (TMA) {
        pl.box = std::min(a.kv.p.page_size, G::TK);
        int r = pa_map(&maps.k, a.kv.p.k, a, pl.box);
        if (r == JYC_OK) r = pa_map(&maps.v, a.kv.p.v, a, pl.box);
        if (r != JYC_OK) return r;
    }
    PaWork w;
    pa_work_bytes<HDP, HEADS, TMA>(sms, static_cast<unsigned char*>(work), &w);
    paged_attention_kernel<HDP, HEADS, TMA><<<ctas, G::WARPS * 32, G::SMEM, s>>>(a, pl, w, maps);
    JYC_LAUNCHED();
    if (tiles <= 1) return JYC_OK;  // an item is one unit: none is split
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kPaJoinWarps * 32);
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    JYC_CUDA(cudaLaunchKernelEx(&cfg, paged_join_kernel<HDP, HEADS, TMA>, a, pl, w));
    JYC_LAUNCHED();
    return JYC_OK;
}

bool aligned16(const void* p, int ld) { return ((uintptr_t)p & 15) == 0 && (ld & 3) == 0; }
bool aligned8(const void* p, const void* q) { return (((uintptr_t)p | (uintptr_t)q) & 7) == 0; }

}  // namespace

// Lanes of a head and quads of a lane by head size; rows in launches of fewer
// than 2^30 warps. f(first row, rows, CTAs, warps that share K or V of a row).
template <class F>
static int row_launches(int rows, int KV, int hd, F f) {
    const int lanes = hd <= 32 ? 8 : hd <= 64 ? 16 : 32, per = kRowUnits * (32 / lanes), chunks = (KV + per - 1) / per;
    const int most = std::max(1, (1 << 30) / (2 * chunks)), warps = kRowThreads / 32;
    for (int r0 = 0; r0 < rows; r0 += most) {
        const int n = std::min(most, rows - r0);
        f(r0, n, (unsigned)(((long long)n * 2 * chunks + warps - 1) / warps), chunks);
        JYC_LAUNCHED();
        if (rows - r0 <= most) break;
    }
    return JYC_OK;
}

int launch_paged_append(const float* K, const float* V, int ld, int rows, int KV, int hd, const int* row_seq,
                        const int* row_pos, const PagedKV& kv, const PagedRope& rope, cudaStream_t s) {
    const bool vec = aligned16(K, ld) && aligned16(V, ld) && aligned8(rope.cos_t, rope.sin_t);
    const auto kernel = hd <= 32    ? paged_append_kernel<8, 1>
                        : hd <= 64  ? paged_append_kernel<16, 1>
                        : hd <= 128 ? paged_append_kernel<32, 1>
                                    : paged_append_kernel<32, 2>;
    return row_launches(rows, KV, hd, [&](int r0, int n, unsigned grid, int chunks) {
        kernel<<<grid, kRowThreads, 0, s>>>(K + (size_t)r0 * ld, V + (size_t)r0 * ld, ld, n, KV, hd,
                                            row_seq ? row_seq + r0 : nullptr, row_pos + r0, shifted(kv, row_seq, r0),
                                            rope, chunks, fast_div(2 * chunks), vec);
    });
}

int launch_paged_read(float* K, float* V, int ld, int rows, int KV, int hd, const int* row_seq, const int* row_pos,
                      const PagedKV& kv, cudaStream_t s) {
    const bool vec = aligned16(K, ld) && aligned16(V, ld);
    const auto kernel = hd <= 32    ? paged_read_kernel<8, 1>
                        : hd <= 64  ? paged_read_kernel<16, 1>
                        : hd <= 128 ? paged_read_kernel<32, 1>
                                    : paged_read_kernel<32, 2>;
    return row_launches(rows, KV, hd, [&](int r0, int n, unsigned grid, int chunks) {
        kernel<<<grid, kRowThreads, 0, s>>>(K + (size_t)r0 * ld, V + (size_t)r0 * ld, ld, n, KV, hd,
                                            row_seq ? row_seq + r0 : nullptr, row_pos + r0, shifted(kv, row_seq, r0),
                                            chunks, fast_div(2 * chunks), vec);
    });
}

// The instantiation of a shape: head size and query heads per unit rounded up,
// and how the rows are copied.
#define PA_CASES(F, TMA, ...)                                                                     \
    do {                                                                                          \
        const int G = H / KV;                                                                     \
        if (hd <= 64) {                                                                           \
            if (G <= 4) return F<64, 4, TMA>(__VA_ARGS__);                                        \
            return G <= 8 ? F<64, 8, TMA>(__VA_ARGS__) : F<64, 16, TMA>(__VA_ARGS__);             \
        }                                                                                         \
        if (hd <= 128) {                                                                          \
            if (G <= 4) return F<128, 4, TMA>(__VA_ARGS__);                                       \
            return G <= 8 ? F<128, 8, TMA>(__VA_ARGS__) : F<128, 16, TMA>(__VA_ARGS__);           \
        }                                                                                         \
        if (hd <= 192) {                                                                          \
            if (G <= 4) return F<192, 4, false>(__VA_ARGS__);                                     \
            return G <= 8 ? F<192, 8, false>(__VA_ARGS__) : F<192, 16, false>(__VA_ARGS__);       \
        }                                                                                         \
        if (G <= 4) return F<256, 4, false>(__VA_ARGS__);                                         \
        return G <= 8 ? F<256, 8, false>(__VA_ARGS__) : F<256, 16, false>(__VA_ARGS__);           \
    } while (0)

template <int HDP, int HEADS, bool TMA>
static size_t pa_workspace(int sms) {
    return pa_work_bytes<HDP, HEADS, TMA>(sms, nullptr, nullptr);
}

size_t paged_attention_workspace(int H, int KV, int hd) {
    const int sms = sm_count();
    if (sms == 0) {
        cuda_fail(cudaErrorNoDevice, "paged attention: device query");
        return 0;
    }
    PA_CASES(pa_workspace, false, sms);
}

int launch_paged_attention(const PagedAttn& a, void* work, cudaStream_t s) {
    const int H = a.H, KV = a.KV, hd = a.hd, sms = sm_count();
    PaPlan pl{};
    pl.qblocks = H / KV > 8 ? (H / KV + 15) / 16 : 1;
    pl.units_row = KV * pl.qblocks;
    pl.wide_q = aligned16(a.Q, a.ldq) && aligned8(a.rope.cos_t, a.rope.sin_t);
    const jyc_kv_pages& p = a.kv.p;
    // 16-byte copies, else 4-byte ones (131072 keys of 8 x 128: 62 us to 142; 64 sequences of 2112 of 8 x 64: 61 to 119)
    pl.wide_copy = hd % 16 == 0 && (((uintptr_t)p.k | (uintptr_t)p.v) & 15) == 0 &&
                   ((p.page_stride | p.pos_stride | p.head_stride) & 15) == 0;
    if (pa_tensor_copies(a, pl.wide_copy)) PA_CASES(pa_launch, true, a, pl, sms, work, s);
    PA_CASES(pa_launch, false, a, pl, sms, work, s);
}

}  // namespace jyc
