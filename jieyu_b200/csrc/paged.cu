// paged.cu — int8 K/V cache in pages: rows are quantised as they are written
// (kv_pack_q8's rule, libs/model_libs/attention/attention_q8.h:20-37), read
// back as fp32, and attended over by one new token per sequence (the score,
// softmax and P.V of attention_q8.h:38-184).
#include "paged.cuh"
#include "ptx.cuh"

#include <cuda.h>

#include <algorithm>
#include <atomic>

namespace jyc {

// Error word of the paged operators (kPagedErr* bits), apart from the decode
// kernel's own, which ends that kernel's waits.
__device__ int g_paged_err;

int* paged_error_word() {
    int* p = nullptr;
    if (cudaGetSymbolAddress(reinterpret_cast<void**>(&p), g_paged_err) != cudaSuccess) return nullptr;
    return p;
}

namespace {

__device__ __forceinline__ void paged_flag(int bit) {
    if ((*(volatile int*)&g_paged_err & bit) == 0) atomicOr(&g_paged_err, bit);
}

// Page id of position `pos` of sequence `seq`, -1 (and the error word) when
// the sequence, the position or the id is out of range.
__device__ __forceinline__ int paged_page(const PagedKV& kv, int seq, int pos) {
    if (seq < 0 || seq >= kv.num_seqs || pos / kv.p.page_size >= kv.table_stride) {
        paged_flag(kPagedErrPos);
        return -1;
    }
    const int page = kv.table[(size_t)seq * kv.table_stride + pos / kv.p.page_size];
    if (page < 0 || page >= kv.p.num_pages) {
        paged_flag(kPagedErrPage);
        return -1;
    }
    return page;
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

// Quad qd (elements 4 qd .. 4 qd + 3: pairs 2 qd, 2 qd + 1) rotated by the
// table rows c, s (rope_pos's rounding: one product rounded, one fused sum).
__device__ __forceinline__ float4 rotate4(float4 x, const float* c, const float* s, int qd) {
    const float c0 = __ldg(c + 2 * qd), c1 = __ldg(c + 2 * qd + 1), s0 = __ldg(s + 2 * qd), s1 = __ldg(s + 2 * qd + 1);
    float4 r;
    r.x = __fmaf_rn(x.x, c0, -__fmul_rn(x.y, s0));
    r.y = __fmaf_rn(x.x, s0, __fmul_rn(x.y, c0));
    r.z = __fmaf_rn(x.z, c1, -__fmul_rn(x.w, s1));
    r.w = __fmaf_rn(x.z, s1, __fmul_rn(x.w, c1));
    return r;
}
__device__ __forceinline__ float amax4(float4 x) {
    return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
}
__device__ __forceinline__ uint32_t pack4(float4 x, float inv) {
    return (uint32_t)(q8_round(x.x, inv) & 255) | ((uint32_t)(q8_round(x.y, inv) & 255) << 8) |
           ((uint32_t)(q8_round(x.z, inv) & 255) << 16) | ((uint32_t)(q8_round(x.w, inv) & 255) << 24);
}

// One warp per (row, kv head, K or V); a lane holds up to two quads.
__global__ void paged_append_kernel(const float* K, const float* V, int ld, int rows, int KV, int hd,
                                    const int* row_seq, const int* row_pos, PagedKV kv, PagedRope rope, bool vec) {
    const int lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (unit >= (long long)rows * KV * 2) return;
    const int i = (int)(unit / (KV * 2)), r = (int)(unit % (KV * 2));
    const int h = r >> 1;
    const bool is_k = (r & 1) == 0;
    const int pos = row_pos[i];
    if (pos < 0) return;
    const int page = paged_page(kv, row_seq ? row_seq[i] : i, pos);
    if (page < 0) return;
    const bool rot = rope.cos_t != nullptr && is_k;
    if (rope.cos_t != nullptr && pos >= rope.len) {
        paged_flag(kPagedErrRope);
        return;
    }
    const int half = hd >> 1, nq = hd >> 2;
    const float* src = (is_k ? K : V) + (size_t)i * ld + (size_t)h * hd;
    float4 x[2];
    float amax = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const int qd = lane + 32 * t;
        if (qd >= nq) continue;
        x[t] = load4(src + 4 * qd, vec);
        if (rot) x[t] = rotate4(x[t], rope.cos_t + (size_t)pos * half, rope.sin_t + (size_t)pos * half, qd);
        amax = fmaxf(amax, amax4(x[t]));
    }
    amax = warp_max(amax);
    const float inv = q8_inv(amax);
    const int slot = pos % kv.p.page_size;
    uint32_t* dst = reinterpret_cast<uint32_t*>((is_k ? kv.p.k : kv.p.v) + paged_off(kv, page, slot, h));
    if (lane == 0) (is_k ? kv.p.ks : kv.p.vs)[paged_soff(kv, page, slot, h)] = q8_scale(amax);
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const int qd = lane + 32 * t;
        if (qd < nq) dst[rot ? rope_slot(2 * qd, half) >> 1 : qd] = pack4(x[t], inv);
    }
}

__global__ void paged_read_kernel(float* K, float* V, int ld, int rows, int KV, int hd, const int* row_seq,
                                  const int* row_pos, PagedKV kv) {
    const int lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (unit >= (long long)rows * KV * 2) return;
    const int i = (int)(unit / (KV * 2)), r = (int)(unit % (KV * 2));
    const int h = r >> 1;
    const bool is_k = (r & 1) == 0;
    const int pos = row_pos[i];
    if (pos < 0) return;
    const int page = paged_page(kv, row_seq ? row_seq[i] : i, pos);
    if (page < 0) return;
    const int slot = pos % kv.p.page_size;
    const int8_t* src = (is_k ? kv.p.k : kv.p.v) + paged_off(kv, page, slot, h);
    const float sc = (is_k ? kv.p.ks : kv.p.vs)[paged_soff(kv, page, slot, h)];
    float* dst = (is_k ? K : V) + (size_t)i * ld + (size_t)h * hd;
    for (int e = lane; e < hd; e += 32) dst[e] = __fmul_rn((float)src[e], sc);
}

// ---------------------------------------------------------------------------
// Attention of one new token per sequence.
//
// out = sum_j p_j vs_j v_j / sum_j p_j, p_j = exp(dot_j (ks_j qs) / sqrt(hd)),
// one pass over the keys with a running reference. In base 2, with vs_j =
// 2^e_j f_j (1 <= f_j < 2): ref = max_j (s_j + e_j) - 13, b_j = 2^(s_j - ref);
// the weights w_j = b_j vs_j are below 2^14 and the largest is at least 2^13,
// so as a pair of fp16 (hi + lo, 22 bits) they neither overflow nor lose a
// small vs that carries all the weight; the denominator adds the b_j.
//
// A step reads sum(len) * KV * (2 hd + 8) bytes and is bound by them, so: work
// is a line of units (a unit: TK keys of one kv head of one sequence), cut into equal runs for all resident warps whatever the lengths; a
// warp keeps its next units in flight in its own ring in shared memory across
// the borders of sequences and has no barrier in its loop. Heads of 64 or 128
// on pages that divide a unit or that units divide come by one tensor copy per
// page, K and V each; other shapes by 16- or 4-byte cp.async.
// Keys are the rows of both products and the (up to 8 or 16) query heads of a
// kv head the columns, so nothing of a tile is padding at 8 heads: S^T = K Q^T
// with mma.m16n8k32 s8 (exact dots), O^T = V^T P^T with mma.m16n8k16 f16 (V is
// exact in fp16), the weights transposed between them by movmatrix. Each
// unit's product starts from zero and is added in fp32 with round to nearest
// (the tensor cores' own sums may truncate).
//
// A run that covers an item (a kv head of a sequence) whole writes its rows of
// out; the others leave (o, ref, l) in the workspace and a second kernel,
// launched early, joins them. The warps of a CTA inside one item are joined in
// shared memory first.

constexpr float kPaShift = 13.0f;
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
template <int N>
__device__ __forceinline__ void pa_copy(uint32_t dst, const void* src) {
    if (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
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
// query columns and unread output columns), E the blocks of 8 query heads of a
// unit.
template <int HDP, int E, bool TMA>
struct PaCfg {
    static constexpr int TK = HDP <= 128 ? 32 : 16;      // keys of a unit
    static constexpr int WARPS = HDP <= 128 ? 12 : 8;    // one CTA per SM
    static constexpr int ST = HDP <= 64 ? 4 : HDP <= 128 ? 2 : 3;
    static constexpr int ROWS = 8 * E;
    static constexpr int VOFF = TK * HDP, SOFF = 2 * TK * HDP, MOFF = SOFF + 8 * TK;
    // K and V; then ks, vs and the valid mask, which the tensor copies' variant keeps in registers. A tensor
    // copy's swizzle goes by the address: stages on 1024 bytes
    static constexpr int STAGE = TMA ? SOFF : MOFF + 16;
    static constexpr int PART = ROWS * (HDP + 2);        // floats of a partial: o, then (ref, l) per row
    static constexpr int FOFF = ST * STAGE;              // the current unit's keys, a float4 each
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
    int tk, warps;  // keys of a unit, warps of a CTA
    bool wide_copy; // 16-byte copies
    int box;        // keys of a tensor copy
    uint32_t div_m; // pos / page_size = pos * div_m >> div_s, for pos < 2^31
    int div_s;
};
// The line cut into runs: worker w starts at w * base + min(w, rest).
struct PaLine {
    long long base, rest, workers;
    int per_cta;  // workers of a CTA
    __device__ __forceinline__ long long start(long long w) const {
        w = min(w, workers);
        return w * base + min(w, rest);
    }
    __device__ __forceinline__ long long worker(long long u) const {  // whose run holds unit u
        const long long big = rest * (base + 1);
        return u < big ? u / (base + 1) : rest + (u - big) / base;
    }
};
// Item that a worker's run starts and another one ends.
struct PaTail {
    long long u0, u1;  // units of the item; u1 == 0: none
    int b, r;
};
struct PaWork {
    PaLine* line;
    PaTail* tail;      // [workers]
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
    const long long each = (U + ctas - 1) / ctas;
    l.per_cta = (int)min((long long)warps, max((long long)kPaFewWarps, each));
    l.workers = min((long long)ctas * l.per_cta, U);
    l.base = l.workers ? U / l.workers : 0;
    l.rest = l.workers ? U % l.workers : 0;
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
__device__ __forceinline__ void pa_next(const PagedAttn& a, const PaPlan& pl, PaCursor& c) {
    if (++c.t < c.nt) return;
    c.t = 0;
    if (++c.r < pl.units_row) return;
    c.r = 0;
    c.b++;
    pa_seek(a, pl.tk, c);
}

// A wait that did not end at once: gives up after 2^31 SM cycles (about a
// second) and sets the error word; the unit then counts for nothing.
__device__ __noinline__ bool pa_wait(uint64_t* bar, uint32_t parity) {
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity))
        if (clock64() - t0 > (1LL << 31)) {
            paged_flag(kPagedErrWait);
            return false;
        }
    return true;
}
// box of a map's tensor [page][slot][kv head][dim] -> shared memory (this CTA's)
__device__ __forceinline__ void pa_tensor_copy(uint32_t dst, const CUtensorMap* map, int h, int slot, int page,
                                               uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(map), "r"(0), "r"(h), "r"(slot), "r"(page), "r"(smem_u32(bar))
        : "memory");
}

template <int HDP, int E, bool TMA>
__global__ void __launch_bounds__(PaCfg<HDP, E, TMA>::WARPS * 32, 1)
    paged_attention_kernel(PagedAttn a, PaPlan pl, PaWork work, const __grid_constant__ PaMaps maps) {
    using G = PaCfg<HDP, E, TMA>;
    constexpr int TK = G::TK, ST = G::ST, WARPS = G::WARPS, ROWS = G::ROWS;
    constexpr int NK = HDP / 32, NM = TK / 16, ND = HDP / 16;
    extern __shared__ __align__(128) unsigned char pa_raw[];
    unsigned char* const pa_sm = TMA ? pa_raw + (-smem_u32(pa_raw) & 1023u) : pa_raw;
    __shared__ __align__(8) uint64_t s_bar[WARPS][ST];
    __shared__ long long s_scan[WARPS];
    __shared__ PaCursor s_cur[WARPS];
    __shared__ long long s_first[WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int B = a.kv.num_seqs, group = a.H / a.KV, hd = TMA ? HDP : a.hd;
    griddep_launch();
    if (TMA && lane == 0) {
        for (int i = 0; i < ST; i++) mbar_init(&s_bar[warp][i], 1);
        mbar_fence_init();
    }

    // where the units of each sequence lie in the line
    const int per = (B + WARPS * 32 - 1) / (WARPS * 32);
    const int bs = min(B, tid * per), be = min(B, bs + per);
    long long mine = 0;
    for (int b = bs; b < be; b++) mine += (pa_len(a, b) + TK - 1) / TK;
    mine *= pl.units_row;
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    long long U = 0, ex = incl - mine;
    for (int w = 0; w < WARPS; w++) {
        if (w < warp) ex += s_scan[w];
        U += s_scan[w];
    }
    const PaLine line = pa_line(U, gridDim.x, WARPS);
    if (blockIdx.x == 0 && tid == 0) *work.line = line;
    const long long w0 = (long long)blockIdx.x * line.per_cta;
    for (int w = 0; w < line.per_cta; w++) {
        const long long u = line.start(w0 + w);
        if (u < ex || u >= ex + mine) continue;
        long long at = ex;
        for (int b = bs; b < be; b++) {
            const int len = pa_len(a, b), nt = (len + TK - 1) / TK;
            const long long n = (long long)nt * pl.units_row;
            if (u < at + n) {
                const int k = (int)(u - at);
                s_cur[w] = PaCursor{b, k / nt, k % nt, nt, len};
                s_first[w] = u - k % nt;  // first unit of the item that the run starts in
                break;
            }
            at += n;
        }
    }
    // sequences without a key: rows of zeros
    for (int b = blockIdx.x; b < B; b += gridDim.x)
        if (pa_len(a, b) == 0)
            for (int e = tid; e < a.H * hd; e += WARPS * 32) a.out[(size_t)b * a.ldo + e] = 0.0f;
    __syncthreads();

    const bool worker = warp < line.per_cta;
    const long long u0 = line.start(w0 + warp), u1 = line.start(w0 + warp + 1);
    const long long c0 = line.start(w0), c1 = line.start(w0 + line.per_cta);
    const int count = worker ? (int)(u1 - u0) : 0;
    unsigned char* ring = pa_sm + warp * G::RING;
    const uint32_t ring_a = smem_u32(ring);
    PaCursor cur = PaCursor{0, 0, 0, 0, 0};
    long long item0 = 0;
    if (count > 0) {
        cur = s_cur[warp];
        item0 = s_first[warp];
    }
    // every worker of the CTA inside one item: joined below
    bool joint = false, whole = false;  // whole: and they are all of it
    if (c1 > c0) {
        const long long first = s_first[0], end = first + s_cur[0].nt;
        joint = c1 <= end;
        whole = c0 == first && c1 == end;
    }
    if (worker && lane == 0) work.tail[w0 + warp].u1 = 0;

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
                const int idx = (int)(((unsigned long long)pos * pl.div_m) >> pl.div_s);
                slot = pos - idx * a.kv.p.page_size;
                pg = __ldg(a.kv.table + (size_t)nx.b * a.kv.table_stride + idx);
                ok = true;
            }
            pa_next(a, pl, nx);
        }
        issued++;
    };
    float ksq[ST - 1], vsq[ST - 1];
    bool inq[ST - 1];
    constexpr int LPR = HDP <= 64 ? 4 : HDP <= 128 ? 8 : 16, RPI = 32 / LPR;  // lanes per row, rows per step
    const int cc = (lane & (LPR - 1)) * 16, cr = lane / LPR;
    const int8_t* const kcol = a.kv.p.k + cc;
    const int8_t* const vcol = a.kv.p.v + cc;
    auto issue = [&](int st) {  // copies of the unit that was looked up last
        if (ok && (unsigned)pg >= (unsigned)a.kv.p.num_pages) {
            paged_flag(kPagedErrPage);
            ok = false;
        }
        if constexpr (TMA) {
            // the scales of the units in flight wait in registers (lane j: key j)
#pragma unroll
            for (int i = 0; i + 1 < ST - 1; i++) {
                ksq[i] = ksq[i + 1];
                vsq[i] = vsq[i + 1];
                inq[i] = inq[i + 1];
            }
            ksq[ST - 2] = vsq[ST - 2] = 0.0f;
            inq[ST - 2] = ok;
            const bool lead = ok && (lane & (pl.box - 1)) == 0;
            const unsigned leads = __ballot_sync(0xffffffffu, lead);
            if (lane == 0) mbar_expect_tx(&s_bar[warp][st], __popc(leads) * pl.box * (2 * HDP));
            __syncwarp();
            if (lead) {
                const uint32_t dst = ring_a + st * G::STAGE + lane * HDP;
                pa_tensor_copy(dst, &maps.k, h, slot, pg, &s_bar[warp][st]);
                pa_tensor_copy(dst + G::VOFF, &maps.v, h, slot, pg, &s_bar[warp][st]);
            }
            if (ok) {
                const long long so = (long long)pg * a.kv.p.spage_stride + (long long)slot * a.kv.p.spos_stride + hsoff;
                ksq[ST - 2] = __ldg(a.kv.p.ks + so);
                vsq[ST - 2] = __ldg(a.kv.p.vs + so);
            }
            return;
        }
        const uint32_t base = ring_a + st * G::STAGE;
        const unsigned mask = __ballot_sync(0xffffffffu, ok);
        long long off = 0;
        if (ok) {
            off = (long long)pg * a.kv.p.page_stride + (long long)slot * a.kv.p.pos_stride + hoff;
            const long long so = (long long)pg * a.kv.p.spage_stride + (long long)slot * a.kv.p.spos_stride + hsoff;
            pa_copy<4>(base + G::SOFF + 4 * lane, a.kv.p.ks + so);
            pa_copy<4>(base + G::SOFF + 4 * TK + 4 * lane, a.kv.p.vs + so);
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
                    pa_copy<16>(dst, kcol + o);
                    pa_copy<16>(dst + G::VOFF, vcol + o);
                }
            }
        } else {
            for (int row = 0; row < TK; row++) {
                const long long o = __shfl_sync(0xffffffffu, off, row);
                if (!((mask >> row) & 1)) continue;
                for (int c = lane; c * 4 < hd; c += 32) {
                    const uint32_t dst = base + G::at(row, c / 4) + (c & 3) * 4;
                    pa_copy<4>(dst, a.kv.p.k + o + c * 4);
                    pa_copy<4>(dst + G::VOFF, a.kv.p.v + o + c * 4);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    lookup();
#pragma unroll
    for (int i = 0; i < ST - 1; i++) {
        issue(i);
        lookup();
    }

    // lane (g, t): query head g (and g + 8) as B fragments, bytes 4 t .. 4 t + 3 of every 16; of the results the
    // heads 2 t, 2 t + 1 (and 8 more), for which it keeps the reference, its share of the sum, and the dims 2 g,
    // 2 g + 1 of every 16
    uint32_t qf[NK][E][2];
    float qsl[E][2], ref[E][2], l[E][2], o[ND][E][4];
    bool fresh = true;
    int st = 0;
    uint32_t phase = 0u;
    const float up = __fmul_rn(a.scale, 1.44269504088896341f);

    for (int n = 0; n < count; n++) {
        if (fresh) {
            // the item's query heads: rotated and quantised per head
            fresh = false;
            const int qb = cur.r % pl.qblocks, kvh = cur.r / pl.qblocks;
            const int half = hd >> 1;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int row = qb * ROWS + 8 * e + g;
                const bool live = row < group;
                const float* q = a.Q + (size_t)cur.b * a.ldq + (size_t)(kvh * group + (live ? row : 0)) * hd;
                const size_t tp = (size_t)(cur.len - 1) * half;
                float4 x[2 * NK];
                float amax = 0.0f;
#pragma unroll
                for (int i = 0; i < 2 * NK; i++) {
                    int src = 4 * i + t;  // quad stored in slot 4 i + t
                    x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (!live || 4 * src >= hd) continue;
                    if (a.rope.cos_t) {
                        src = rope_slot(2 * src, half) >> 1;  // its own inverse
                        x[i] = rotate4(load4(q + 4 * src, false), a.rope.cos_t + tp, a.rope.sin_t + tp, src);
                    } else {
                        x[i] = load4(q + 4 * src, false);
                    }
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
        // the next unit's copies go to the stage that the last iteration read
        __syncwarp();
        bool in = false;
        float kscale = 0.0f, vscale = 0.0f;
        if constexpr (TMA) {
            in = inq[0];
            kscale = ksq[0];
            vscale = vsq[0];
        }
        issue(st == 0 ? ST - 1 : st - 1);
        lookup();
        if constexpr (TMA) {
            if (!mbar_try_wait(&s_bar[warp][st], phase) && !pa_wait(&s_bar[warp][st], phase)) in = false;
        } else {
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
            keys[lane] = in ? make_float4(kscale, 0.0f, (float)ex, vscale) : make_float4(0.0f, -INFINITY, 0.0f, 0.0f);
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
        // weights, transposed into B fragments: head g, keys 16 m + 2 t, + 1 and 8 later
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
                    hi[m][e][i] = pa_transpose(ph);
                    lo[m][e][i] = pa_transpose(pa_pack(w0 - hf.x, w1 - hf.y));
                }
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
                        pa_mma_f16(vf, lo[m][e], c[i][e]);
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
        if (++st == ST) {
            st = 0;
            phase ^= 1u;
        }

        const bool item_end = cur.t == cur.nt - 1;
        if (!item_end && n + 1 < count) {
            cur.t++;
            continue;
        }
        // the end of an item or of the run
#pragma unroll
        for (int e = 0; e < E; e++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[e][j] += __shfl_xor_sync(0xffffffffu, l[e][j], x);
        const bool from_start = item0 >= u0;
        if (from_start && item_end) {
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
            if (from_start && lane == 0 && !whole)
                work.tail[w0 + warp] = PaTail{item0, item0 + cur.nt, cur.b, cur.r};
            if (joint) break;  // o, ref and l stay in registers
            float* part = work.part + ((size_t)(w0 + warp) * 2 + (from_start ? 1 : 0)) * G::PART;
#pragma unroll
            for (int e = 0; e < E; e++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int row = 8 * e + 2 * t + j;
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
            pa_next(a, pl, cur);
            fresh = true;
        }
    }
    if (!TMA) asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (!joint || (whole && line.start(w0 + 1) == c1)) return;

    // join the CTA's workers (their rings are free now)
    float* buf = reinterpret_cast<float*>(ring);
    if (worker)
#pragma unroll
        for (int e = 0; e < E; e++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int row = 8 * e + 2 * t + j;
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
    float* part = work.part + ((size_t)w0 * 2 + (c0 == s_first[0] ? 1 : 0)) * G::PART;
    for (int i = tid; i < ROWS * HDP / 4; i += WARPS * 32) {
        const int row = i / (HDP / 4), d = i % (HDP / 4) * 4;
        float M = kPaLow, L = 0.0f;
        float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < line.per_cta; w++)
            M = fmaxf(M, reinterpret_cast<const float*>(pa_sm + w * G::RING)[ROWS * HDP + 2 * row]);
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

// The items that start in one worker's run and end in another's: a CTA per
// worker. The parts of an item are, in order, those of single workers at its
// ends and one of every CTA inside it; warp w adds parts w, w + 8, ... for RB
// query rows at a time (every load of a part in flight at once), then the
// warps' sums are joined in shared memory.
constexpr int kPaJoinWarps = 8;
template <int HDP, int E, bool TMA>
__global__ void __launch_bounds__(kPaJoinWarps * 32) paged_join_kernel(PagedAttn a, PaPlan pl, PaWork work) {
    using G = PaCfg<HDP, E, TMA>;
    constexpr int ROWS = G::ROWS, NV = (HDP + 127) / 128, RB = HDP <= 128 ? 8 : 4;
    __shared__ __align__(16) float s_o[kPaJoinWarps][RB][HDP];
    __shared__ float2 s_rl[kPaJoinWarps][RB];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = a.H / a.KV, hd = a.hd;
    const long long wf = blockIdx.x;
    griddep_wait();
    const PaLine line = *work.line;
    if (wf >= line.workers) return;
    const PaTail tail = work.tail[wf];
    if (tail.u1 == 0) return;
    const long long wl = line.worker(tail.u1 - 1);
    const int per = line.per_cta, cf = (int)(wf / per), cl = (int)(wl / per);
    auto inside = [&](long long c) { return line.start(c * per) >= tail.u0 && line.start((c + 1) * per) <= tail.u1; };
    const int na = inside(cf) ? 1 : (int)(min(wl, (long long)cf * per + per - 1) - wf) + 1;
    const int nm = max(0, cl - cf - 1), nb = cl == cf ? 0 : inside(cl) ? 1 : (int)(wl - (long long)cl * per) + 1;
    const int np = na + nm + nb;
    const int qb = tail.r % pl.qblocks, kvh = tail.r / pl.qblocks;
    for (int r0 = 0; r0 < ROWS && qb * ROWS + r0 < group; r0 += RB) {
        const int rows = min(RB, group - qb * ROWS - r0);
        float4 o[RB][NV];
        float ref = kPaLow, l = 0.0f;  // of row lane % RB
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll
            for (int d = 0; d < NV; d++) o[r][d] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = warp; i < np; i += kPaJoinWarps) {
            const int w = i < na ? (int)wf + i : i < na + nm ? (cf + 1 + i - na) * per : cl * per + (i - na - nm);
            const float* p = work.part + ((size_t)w * 2 + (i == 0 ? 1 : 0)) * G::PART;
            const float2 rl = *reinterpret_cast<const float2*>(p + ROWS * HDP + 2 * (r0 + (lane & (RB - 1))));
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
        __syncthreads();  // the last row block's sums are read
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll
            for (int d = 0; d < NV; d++)
                if (128 * d + 4 * lane < HDP) *reinterpret_cast<float4*>(&s_o[warp][r][128 * d + 4 * lane]) = o[r][d];
        if (lane < RB) s_rl[warp][lane] = make_float2(ref, l);
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

// SMs of the current device (0: no device).
int sm_count() {
    static std::atomic<int> sms[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (dev < 64 && (n = sms[dev].load(std::memory_order_relaxed)) > 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    if (dev < 64) sms[dev].store(n, std::memory_order_relaxed);
    return n;
}

size_t align16(size_t n) { return (n + 15) / 16 * 16; }

template <int HDP, int E, bool TMA>
size_t pa_work_bytes(int ctas, unsigned char* base, PaWork* w) {
    const size_t workers = (size_t)ctas * PaCfg<HDP, E, TMA>::WARPS;
    const size_t head = align16(sizeof(PaLine)), at = align16(workers * sizeof(PaTail));
    if (w) *w = PaWork{reinterpret_cast<PaLine*>(base), reinterpret_cast<PaTail*>(base + head),
                       reinterpret_cast<float*>(base + head + at)};
    return head + at + workers * 2 * PaCfg<HDP, E, TMA>::PART * sizeof(float);
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
    const CUresult r = reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(fn)(
        m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, base, dims, strides, boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
        a.hd == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return cuda_fail(cudaErrorInvalidValue, "cuTensorMapEncodeTiled");
    return JYC_OK;
}

// Tensor copies need rows of 64 or 128 bytes, strides below 2^40 that are multiples of 16 bytes, pages that
// a unit of 32 keys fills or that fill a unit, and boxes that start on 128 bytes of shared memory.
bool pa_tensor_copies(const PagedAttn& a, bool aligned) {
    const jyc_kv_pages& p = a.kv.p;
    const long long far = std::max(p.page_stride, std::max(p.pos_stride, p.head_stride));
    const bool nonzero = (p.head_stride > 0 || a.KV == 1) && (p.pos_stride > 0 || p.page_size == 1) &&
                         (p.page_stride > 0 || p.num_pages == 1);
    return aligned && nonzero && far < (1LL << 40) && (a.hd == 64 || a.hd == 128) &&
           (p.page_size % 32 == 0 || (32 % p.page_size == 0 && p.page_size * a.hd % 128 == 0));
}

template <int HDP, int E, bool TMA>
int pa_launch(const PagedAttn& a, PaPlan pl, int sms, void* work, cudaStream_t s) {
    using G = PaCfg<HDP, E, TMA>;
    // the attribute belongs to the device
    static std::atomic<bool> ready[64];
    int dev = 0;
    JYC_CUDA(cudaGetDevice(&dev));
    if (dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {
        JYC_CUDA(cudaFuncSetAttribute(paged_attention_kernel<HDP, E, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      G::SMEM));
        if (dev < 64) ready[dev].store(true, std::memory_order_release);
    }
    const long long cap = (long long)a.kv.table_stride * a.kv.p.page_size, tiles = (cap + G::TK - 1) / G::TK;
    const long long items = (long long)a.kv.num_seqs * pl.units_row;
    // no more CTAs than the longest possible lengths have units for
    const long long units = tiles >= (1LL << 31) / items ? 1LL << 31 : items * tiles;
    const int ctas = (int)std::max(1LL, std::min((long long)sms, (units + kPaFewWarps - 1) / kPaFewWarps));
    pl.tk = G::TK;
    pl.warps = G::WARPS;
    PaMaps maps{};
    if (TMA) {
        pl.box = std::min(a.kv.p.page_size, G::TK);
        int r = pa_map(&maps.k, a.kv.p.k, a, pl.box);
        if (r == JYC_OK) r = pa_map(&maps.v, a.kv.p.v, a, pl.box);
        if (r != JYC_OK) return r;
    }
    PaWork w;
    pa_work_bytes<HDP, E, TMA>(sms, static_cast<unsigned char*>(work), &w);
    paged_attention_kernel<HDP, E, TMA><<<ctas, G::WARPS * 32, G::SMEM, s>>>(a, pl, w, maps);
    JYC_LAUNCHED();
    if (tiles <= 1) return JYC_OK;  // an item is one unit: none is split
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas * G::WARPS);
    cfg.blockDim = dim3(kPaJoinWarps * 32);
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    JYC_CUDA(cudaLaunchKernelEx(&cfg, paged_join_kernel<HDP, E, TMA>, a, pl, w));
    JYC_LAUNCHED();
    return JYC_OK;
}

bool aligned16(const void* p, int ld) { return ((uintptr_t)p & 15) == 0 && (ld & 3) == 0; }

}  // namespace

int launch_paged_append(const float* K, const float* V, int ld, int rows, int KV, int hd, const int* row_seq,
                        const int* row_pos, const PagedKV& kv, const PagedRope& rope, cudaStream_t s) {
    const long long units = (long long)rows * KV * 2;
    if (units == 0) return JYC_OK;
    paged_append_kernel<<<(unsigned)((units + 7) / 8), 256, 0, s>>>(K, V, ld, rows, KV, hd, row_seq, row_pos, kv, rope,
                                                                    aligned16(K, ld) && aligned16(V, ld));
    JYC_LAUNCHED();
    return JYC_OK;
}

int launch_paged_read(float* K, float* V, int ld, int rows, int KV, int hd, const int* row_seq, const int* row_pos,
                      const PagedKV& kv, cudaStream_t s) {
    const long long units = (long long)rows * KV * 2;
    if (units == 0) return JYC_OK;
    paged_read_kernel<<<(unsigned)((units + 7) / 8), 256, 0, s>>>(K, V, ld, rows, KV, hd, row_seq, row_pos, kv);
    JYC_LAUNCHED();
    return JYC_OK;
}

// The instantiation of a shape: head size rounded up, two blocks of 8 query
// heads per unit above 8, and how the rows are copied.
#define PA_CASES(F, TMA, ...)                                                                   \
    do {                                                                                        \
        const bool many = H / KV > 8;                                                           \
        if (hd <= 64) return many ? F<64, 2, TMA>(__VA_ARGS__) : F<64, 1, TMA>(__VA_ARGS__);    \
        if (hd <= 128) return many ? F<128, 2, TMA>(__VA_ARGS__) : F<128, 1, TMA>(__VA_ARGS__); \
        if (hd <= 192) return many ? F<192, 2, false>(__VA_ARGS__) : F<192, 1, false>(__VA_ARGS__); \
        return many ? F<256, 2, false>(__VA_ARGS__) : F<256, 1, false>(__VA_ARGS__);            \
    } while (0)

template <int HDP, int E, bool TMA>
static size_t pa_workspace(int sms) {
    return pa_work_bytes<HDP, E, TMA>(sms, nullptr, nullptr);
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
    // n / d for n < 2^31: with 2^(s-1) < d <= 2^s and m = ceil(2^(31+s) / d), m d - 2^(31+s) < d <= 2^s, so the
    // error of n m / 2^(31+s) is below 2^-31 n < 1 / d at every n; m < 2^32
    int sh = 0;
    while ((1LL << sh) < a.kv.p.page_size) sh++;
    pl.div_s = 31 + sh;
    pl.div_m = (uint32_t)(((1ULL << pl.div_s) + a.kv.p.page_size - 1) / a.kv.p.page_size);
    const jyc_kv_pages& p = a.kv.p;
    pl.wide_copy = hd % 16 == 0 && (((uintptr_t)p.k | (uintptr_t)p.v) & 15) == 0 &&
                   ((p.page_stride | p.pos_stride | p.head_stride) & 15) == 0;
    if (pa_tensor_copies(a, pl.wide_copy)) PA_CASES(pa_launch, true, a, pl, sms, work, s);
    PA_CASES(pa_launch, false, a, pl, sms, work, s);
}

}  // namespace jyc
