// paged.cu — int8 K/V cache in pages: rows are quantised as they are written
// (kv_pack_q8's rule, libs/model_libs/attention/attention_q8.h:20-37), read
// back as fp32, and attended over by one new token per sequence (the score,
// softmax and P.V of attention_q8.h:38-184).
#include "paged.cuh"
#include "paged_line.cuh"
#include "ptx.cuh"
#include "tmap.cuh"

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
    static Entry done[96];
    static std::mutex mu;
    int dev = 0;
    JYC_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lk(mu);
    Entry* e = done;
    while (e < done + 96 && e->kernel && e->kernel != kernel) e++;
    if (e < done + 96 && e->kernel && dev < 64 && (e->devices >> dev & 1)) return JYC_OK;
    JYC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (e < done + 96 && dev < 64) {
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

// bytes 0, 2 (ODD: 1, 3) of x = q ^ 0x80 as the halves q: 0x6400 | u is 1024 + u
template <bool ODD>
__device__ __forceinline__ uint32_t pa_half2(uint32_t x) {
    const uint32_t m = __byte_perm(x, 0x64646464u, ODD ? 0x4341 : 0x4240);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&m), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&r);
}
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

// Sizes of one instantiation: HDP is the head size rounded up (the columns
// behind it hold whatever the ring held, finite as integers; they meet zero
// query columns and unread output columns), HEADS the query heads of a unit.
template <int HDP_, int HEADS, bool TMA>
struct PaCfg {
    using Args = PagedAttn;
    static __device__ __forceinline__ int len(const PagedAttn& a, int b) { return pa_len(a, b); }
    static constexpr bool STAT = false, TEAM = false;
    static constexpr int HDP = HDP_;
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
template <int HDP, int HEADS, bool TMA>
__global__ void __launch_bounds__(PaCfg<HDP, HEADS, TMA>::WARPS * 32, 1)
    paged_attention_kernel(PagedAttn a, PaPlan pl, PaWork work, const __grid_constant__ PaMaps maps) {
    using G = PaCfg<HDP, HEADS, TMA>;
    constexpr int TK = G::TK, ST = G::ST, WARPS = G::WARPS, ROWS = G::ROWS, E = G::E;
    constexpr int NK = HDP / 32, NM = TK / 16, ND = HDP / 16;
    extern __shared__ __align__(128) unsigned char pa_raw[];
    unsigned char* const pa_sm = TMA ? pa_raw + (-smem_u32(pa_raw) & 1023u) : pa_raw;
    __shared__ __align__(8) uint64_t s_bar[WARPS][ST][2];  // K, V
    __shared__ PaShared<G> sh;
    const uint64_t policy = policy_evict_first();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int group = a.H / a.KV, hd = TMA ? HDP : a.hd;
    griddep_launch();
    if (TMA && lane == 0) {
        if (warp == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.k) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.v) : "memory");
        }
        for (int i = 0; i < 2 * ST; i++) mbar_init(&s_bar[warp][0][i], 1);
        mbar_fence_init();
    }

    const PaRun run = pa_start<G>(a, pl, sh, hd);
    const long long w0 = run.w0, u0 = run.u0;
    const bool joint = run.joint, alone = run.alone;
    const int step = run.step;
    int count = run.count;
    PaCursor cur = run.cur;
    long long item0 = run.item0;
    unsigned char* ring = pa_sm + warp * G::RING;
    const uint32_t ring_a = smem_u32(ring);
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
            pa_next<G>(a, pl, nx, step);
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
            if (!pa_wait(&s_bar[warp][st][0], phase, &g_paged_err)) gave_up = true;
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
            if (!pa_wait(&s_bar[warp][st][1], phase, &g_paged_err)) gave_up = true;
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
            pa_finish<G>(a, pl, work, cur, hd, o, ref, l);
        } else {
            if (joint) break;  // o, ref and l stay in registers
            tail = from_start;
            pa_store<G>(work.part + ((size_t)(w0 + warp) * 2 + (from_start ? 1 : 0)) * G::PART, true, o, ref, l);
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
            pa_wait(&s_bar[warp][st][0], phase, &g_paged_err);
            pa_wait(&s_bar[warp][st][1], phase, &g_paged_err);
            if (++st == ST) {
                st = 0;
                phase ^= 1u;
            }
        }
    pa_end<G>(a, pl, work, sh, run, count, cur, item0, tail, pa_sm, hd, o, ref, l);
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
    if (w) *w = PaWork{reinterpret_cast<PaTail*>(base), reinterpret_cast<float*>(base + at), nullptr};
    return at + workers * 2 * PaCfg<HDP, HEADS, TMA>::PART * sizeof(float);
}

// Map of a cache array as [page][slot][kv head][dim], boxes of `box` slots of one head.
int pa_map(CUtensorMap* m, int8_t* base, const PagedAttn& a, int box) {
    void* fn = nullptr;
    if (int e = tensor_map_encoder(&fn)) return e;
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
    JYC_CUDA(cudaLaunchKernelEx(&cfg, paged_join_kernel<G>, a, pl, w));
    JYC_LAUNCHED();
    return JYC_OK;
}

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
