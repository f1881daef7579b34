// i8.cu — C = (A W^T) * (a_scale w_scale) + bias over 8-bit integers with 32-bit sums, and the rows of
// fp32 activations in 8 bits that go into it (kv_pack_q8's rule over a whole row,
// libs/model_libs/attention/attention_q8.h:24-35).
//
// The products run on tcgen05.mma kind::i8: M = 128 output channels, so that neighbouring lanes of the
// accumulator are neighbouring columns of C (a warp stores 128 contiguous bytes of a row straight from tensor
// memory, no pass through shared memory), N = a tile of tokens, K in chunks of 128 bytes brought by tensor copies
// (TMA) in the 128-byte swizzle that the products read. Copies fill what lies outside of A, W and k with zeros, so edges
// need no care but at the stores. Whole-number sums are exact, so K may be split in any way with the same result.
//
// Measured, with the rows' quantising: 4096 tokens of 14336 x 4096 219 us, of them 17 quantising (the product alone 177 us
// back to back, 2.7 P operations a second; 151 without its stores, 140 without copies and stores, 13 rounds of tiles where
// 12.1 would do); 48 tokens of 14336 x 4090 22 us (floor 9.5), one token of 4096 x 4096 12 us (floor 2.6): two launches and
// the first and last steps of a CTA (tensor memory, first copies, results) are half of it.
#include "i8.cuh"
#include "follow.cuh"
#include "kernels.cuh"
#include "mega.cuh"
#include "paged.cuh"
#include "ptx.cuh"
#include "tc.cuh"
#include "tmap.cuh"

#include <algorithm>

namespace jyc {

namespace {

constexpr int kQrThreads = 256;

// A CTA quantises one row: its maximum, then its values. A thread holds up to QUADS quads of the row in registers, all
// requested at once (QUADS 0: rows that are longer, or do not lie on 16 bytes, are read again, value by value: 4096 rows of
// 4090 values 27 us, 20 where rows lie on 16 bytes; 1024 rows of 20000 43 us, of 16384 25).
template <int QUADS>
__global__ void __launch_bounds__(kQrThreads) quantize_rows_kernel(const float* x, int ldx, int k, int8_t* q, int ldq,
                                                                   float* scale) {
    __shared__ float s_max[kQrThreads / 32];
    const int tid = threadIdx.x;
    griddep_wait();
    griddep_launch();  // a product that follows may prepare itself
    const float* row = x + (size_t)blockIdx.x * ldx;
    int8_t* to = q + (size_t)blockIdx.x * ldq;
    float amax = 0.0f;
    float4 v[QUADS > 0 ? QUADS : 1];
    if constexpr (QUADS > 0) {
#pragma unroll
        for (int i = 0; i < QUADS; i++) {
            const int at = 4 * (tid + i * kQrThreads);
            v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (at + 3 < k)
                v[i] = __ldg(reinterpret_cast<const float4*>(row + at));
            else if (at < k) {
                v[i].x = __ldg(row + at);
                if (at + 1 < k) v[i].y = __ldg(row + at + 1);
                if (at + 2 < k) v[i].z = __ldg(row + at + 2);
            }
        }
#pragma unroll
        for (int i = 0; i < QUADS; i++)
            amax = fmaxf(amax, fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w))));
    } else {
        for (int i = tid; i < k; i += kQrThreads) amax = fmaxf(amax, fabsf(__ldg(row + i)));
    }
    amax = warp_max(amax);
    if ((tid & 31) == 0) s_max[tid >> 5] = amax;
    __syncthreads();
    for (int w = 0; w < kQrThreads / 32; w++) amax = fmaxf(amax, s_max[w]);
    const float inv = q8_inv(amax);
    if (tid == 0) scale[blockIdx.x] = q8_scale(amax);
    if constexpr (QUADS > 0) {
#pragma unroll
        for (int i = 0; i < QUADS; i++) {
            const int at = 4 * (tid + i * kQrThreads);
            const int b[4] = {q8_round(v[i].x, inv), q8_round(v[i].y, inv), q8_round(v[i].z, inv), q8_round(v[i].w, inv)};
            if (at + 3 < k)
                *reinterpret_cast<uint32_t*>(to + at) =
                    __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
            else
#pragma unroll
                for (int e = 0; e < 3; e++)
                    if (at + e < k) to[at + e] = (int8_t)b[e];
        }
    } else {
        for (int i = tid; i < k; i += kQrThreads) to[i] = (int8_t)q8_round(__ldg(row + i), inv);
    }
}

// ---------------------------------------------------------------------------
constexpr int kErrI8 = 10;     // device error word: a bounded wait gave up
constexpr int kI8Rows = 128;   // output channels of a tile
constexpr int kI8Chunk = 128;  // bytes of K of a stage
constexpr int kI8Threads = 192;  // copies, products, four warps of results

// D[tmem] (+)= A[smem] . B[smem]^T, signed bytes, 32-bit sums
__device__ __forceinline__ void i8_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// 32-bit sums, signed bytes, both K-major, M = 128
__device__ __forceinline__ constexpr uint32_t i8_idesc(int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kI8Rows >> 4) << 24);
}
// box of a map's tensor [row][k] -> shared memory (this CTA's)
__device__ __forceinline__ void i8_copy(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}
// 16 columns of this warp's 32 lanes
__device__ __forceinline__ void i8_tmem_ld16(uint32_t ta, int* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(ta)
        : "memory");
}
__device__ __forceinline__ void i8_tmem_ld32(uint32_t ta, int* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(ta)
        : "memory");
}
__device__ __forceinline__ void i8_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Sum, scales and bias: one rounding each.
__device__ __forceinline__ float i8_out(int sum, float as, float ws, bool add, float bias) {
    const float v = __fmul_rn(__int2float_rn(sum), __fmul_rn(as, ws));
    return add ? __fadd_rn(v, bias) : v;
}

// N tokens of this lane's channel, all of which exist
template <int N, bool BIAS>
__device__ __forceinline__ void i8_store(const int* v, const float* as, float ws, float bias, float* to, int ldc) {
#pragma unroll
    for (int u = 0; u < N; u += 4) {
        const float4 a = *reinterpret_cast<const float4*>(as + u);
        __stcs(to, i8_out(v[u], a.x, ws, BIAS, bias));
        __stcs(to += ldc, i8_out(v[u + 1], a.y, ws, BIAS, bias));
        __stcs(to += ldc, i8_out(v[u + 2], a.z, ws, BIAS, bias));
        __stcs(to += ldc, i8_out(v[u + 3], a.w, ws, BIAS, bias));
        to += ldc;
    }
}
// This warp's 32 channels of `live` tokens from tensor memory at ta, N at a time, to C; as: the tokens' scales in shared
// memory. (One warp a scheduler at 20 instructions a result was what bounded the large product: 217 us, 177 with eight
// warps and this form.)
template <int N>
__device__ __forceinline__ void i8_results(const I8Gemm& g, uint32_t ta, const float* as, int live, int j, float* to) {
    const bool col = j < g.n, all = __all_sync(0xffffffffu, col);
    const float ws = col ? __ldg(g.ws + j) : 0.0f, bias = col && g.bias ? __ldg(g.bias + j) : 0.0f;
#pragma unroll 1
    for (int c = 0; c < live; c += N) {
        int v[N];
        if constexpr (N == 32)
            i8_tmem_ld32(ta + c, v);
        else
            i8_tmem_ld16(ta + c, v);
        if (c + N <= live && all) {
            if (g.bias)
                i8_store<N, true>(v, as + c, ws, bias, to, g.ldc);
            else
                i8_store<N, false>(v, as + c, ws, bias, to, g.ldc);
            to += (size_t)N * g.ldc;
            continue;
        }
#pragma unroll
        for (int u = 0; u < N; u++, to += g.ldc)
            if (col && c + u < live) *to = i8_out(v[u], as[c + u], ws, g.bias != nullptr, bias);
    }
}

// four sums of CTA `rank` of the cluster at the address that they have here
__device__ __forceinline__ int4 i8_far(uint32_t at, int rank) {
    uint32_t far;
    int4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(far) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(far)
                 : "memory");
    return v;
}

struct I8Maps {
    CUtensorMap w, a;
};

__device__ __forceinline__ void i8_prefetch(const I8Maps& maps) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.w) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.a) : "memory");
}

// Bounded waits of one CTA: after any of them gave up, every later one is skipped.
struct I8Wait {
    int* err;
    volatile int* abort;
    __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t parity) const {
        if (mbar_try_wait(bar, parity)) return true;
        if (*abort) return false;
        if (mbar_wait_err(bar, parity, err, kErrI8)) return true;
        *abort = 1;
        return false;
    }
};

// Many tiles: a pair of CTAs (a cluster of 2) takes every pair-count-th tile of 256 channels x 256 tokens, tokens first.
// Each CTA holds 128 of the channels and copies 128 of the tokens; the pair's products (cta_group::2, issued by the first
// CTA) read both halves of the tokens, so that a CTA brings 32 KB for what one alone would need 48 KB for. Two
// accumulators: a tile's results leave while the next one's products run.
constexpr int kI8PairTokens = 256, kI8PairStages = 6, kI8PairThreads = 320;
constexpr int kI8PairStage = (kI8Rows + kI8PairTokens / 2) * kI8Chunk, kI8PairSmem = 1024 + kI8PairStages * kI8PairStage;

__device__ __forceinline__ void i8_pair_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// arrives on `bar` of both CTAs when every product this thread issued so far has completed
__device__ __forceinline__ void i8_pair_commit(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}
// address of the first CTA's copy of a shared variable
__device__ __forceinline__ uint32_t i8_lead(const void* p) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(smem_u32(p)));
    return at;
}
// box -> this CTA's shared memory, its bytes counted by the first CTA's barrier
__device__ __forceinline__ void i8_pair_copy(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

__global__ void __launch_bounds__(kI8PairThreads, 1) i8_pair_kernel(I8Gemm g, const __grid_constant__ I8Maps maps, int* err) {
    constexpr int BN = kI8PairTokens, ST = kI8PairStages;
    constexpr uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(2 * kI8Rows >> 4) << 24);
    extern __shared__ unsigned char i8_raw[];
    __shared__ __align__(8) uint64_t full[ST], empty[ST], accf[2], acce[2];  // full and acce: the first CTA's are used
    __shared__ uint32_t s_tmem;
    __shared__ __align__(16) float s_as[8][BN / 2];
    __shared__ int s_abort;
    unsigned char* const sm = i8_raw + (-smem_u32(i8_raw) & 1023u);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = blockIdx.x & 1, pairs = gridDim.x >> 1;
    const int tt = (g.m + BN - 1) / BN, tiles = (g.n + 2 * kI8Rows - 1) / (2 * kI8Rows) * tt;
    const int nch = (g.k + kI8Chunk - 1) / kI8Chunk;
    const I8Wait wait{err, &s_abort};
    if (tid == 0) {
        i8_prefetch(maps);
        for (int s = 0; s < ST; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&accf[b], 1);
            mbar_init(&acce[b], 2 * (kI8PairThreads - 64));
        }
        s_abort = 0;
        mbar_fence_init();
    }
    if (warp == 0) {
        __syncwarp();
        tmem_alloc_pair(&s_tmem, 2 * BN);
    }
    tc_fence_before();
    __syncthreads();
    i8_cluster_sync();  // the other CTA's barriers are there
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    griddep_wait();

    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (int tile = blockIdx.x >> 1; ok && tile < tiles; tile += pairs)
                for (int c = 0; c < nch; c++, it++) {
                    const int s = it % ST;
                    if (it >= ST && !(ok = wait(&empty[s], ((it / ST) - 1) & 1))) break;
                    if (rank == 0) mbar_expect_tx(&full[s], 2 * kI8PairStage);
                    const uint32_t bar = i8_lead(&full[s]);
                    unsigned char* const st = sm + s * kI8PairStage;
                    i8_pair_copy(st, &maps.w, c * kI8Chunk, (tile / tt * 2 + rank) * kI8Rows, bar);
                    i8_pair_copy(st + kI8Rows * kI8Chunk, &maps.a, c * kI8Chunk, tile % tt * BN + rank * (BN / 2), bar);
                }
            // no copy may still be landing when the CTAs exit (matters only after an error)
            if (rank == 0)
                for (int j = max(0, it - ST); j < it; j++) mbar_wait_err(&full[j % ST], (j / ST) & 1, err, kErrI8);
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            int it = 0, i = 0;
            bool ok = true;
            for (int tile = blockIdx.x >> 1; ok && tile < tiles; tile += pairs, i++) {
                const int b = i & 1;
                if (i >= 2 && !(ok = wait(&acce[b], ((i >> 1) - 1) & 1))) break;
                tc_fence_after();
                for (int c = 0; c < nch; c++, it++) {
                    const int s = it % ST;
                    if (!(ok = wait(&full[s], (it / ST) & 1))) break;
                    tc_fence_after();
                    const uint32_t st = smem_u32(sm + s * kI8PairStage);
                    const uint64_t w = sw128_desc(st), a = sw128_desc(st + kI8Rows * kI8Chunk);
#pragma unroll
                    for (int k = 0; k < kI8Chunk / 32; k++)  // 32 bytes of K, in 16-byte units
                        i8_pair_mma(tmem + (uint32_t)(BN * b), w + 2 * k, a + 2 * k, idesc, c != 0 || k != 0);
                    i8_pair_commit(&empty[s]);
                }
                if (ok) i8_pair_commit(&accf[b]);
            }
        }
    } else {
        // eight warps: 32 channels and half of the tokens each
        const int q = warp & 3, half = (warp - 2) >> 2;
        float* const as = s_as[warp - 2];
        int i = 0;
        for (int tile = blockIdx.x >> 1; tile < tiles; tile += pairs, i++) {
            const int b = i & 1, j = (tile / tt * 2 + rank) * kI8Rows + 32 * q + lane, t0 = tile % tt * BN + half * (BN / 2);
            __syncwarp();
#pragma unroll
            for (int c = 0; c < BN / 2; c += 32) as[c + lane] = t0 + c + lane < g.m ? __ldg(g.as + t0 + c + lane) : 0.0f;
            __syncwarp();
            if (!__all_sync(0xffffffffu, wait(&accf[b], (i >> 1) & 1))) break;
            tc_fence_after();
            i8_results<32>(g, tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(BN * b + half * (BN / 2)), as,
                           min(BN / 2, g.m - t0), j, g.C + (size_t)t0 * g.ldc + j);
            tc_fence_before();
            const uint32_t bar = i8_lead(&acce[b]);
            asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
        }
    }
    __syncwarp();
    tc_fence_before();
    i8_cluster_sync();  // neither CTA's memory goes while the other one uses it
    if (warp == 0) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc_pair(tmem, 2 * BN);
    }
}

// Few tiles: a CTA computes one tile over one part of K; the parts of a tile are the CTAs of a cluster, which leave
// their sums in shared memory and each add up a share of the tokens.
template <int BN>
struct I8Few {
    static constexpr int kStage = kI8Rows * kI8Chunk + BN * kI8Chunk;
    static constexpr int kStages = 100 * 1024 / kStage > 6 ? 6 : 100 * 1024 / kStage;  // two CTAs per SM
    static constexpr int kCols = BN < 32 ? 32 : BN;
    static constexpr int kSmem = 1024 + kStages * kStage;
    static_assert(BN * kI8Rows * 4 <= kStages * kStage, "the sums fit the stages");
};
template <int BN>
__global__ void __launch_bounds__(kI8Threads) i8_few_kernel(I8Gemm g, const __grid_constant__ I8Maps maps, int* err) {
    using C = I8Few<BN>;
    extern __shared__ unsigned char i8_raw[];
    __shared__ __align__(8) uint64_t full[C::kStages], empty[C::kStages], accf;
    __shared__ uint32_t s_tmem;
    __shared__ __align__(16) float s_as[4][BN];
    __shared__ int s_abort;
    unsigned char* const sm = i8_raw + (-smem_u32(i8_raw) & 1023u);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, parts = gridDim.z, z = blockIdx.z;
    const int chunks = (g.k + kI8Chunk - 1) / kI8Chunk;
    const int c0 = (int)((long long)chunks * z / parts), nch = (int)((long long)chunks * (z + 1) / parts) - c0;  // > 0
    const I8Wait wait{err, &s_abort};
    if (tid == 0) {
        i8_prefetch(maps);
        for (int s = 0; s < C::kStages; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&accf, 1);
        s_abort = 0;
        mbar_fence_init();
    }
    if (warp == 0) {
        __syncwarp();
        tmem_alloc(&s_tmem, C::kCols);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    griddep_wait();

    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            for (; it < nch; it++) {
                const int s = it % C::kStages;
                if (it >= C::kStages && !wait(&empty[s], ((it / C::kStages) - 1) & 1)) break;
                mbar_expect_tx(&full[s], C::kStage);
                i8_copy(sm + s * C::kStage, &maps.w, (c0 + it) * kI8Chunk, blockIdx.x * kI8Rows, &full[s]);
                i8_copy(sm + s * C::kStage + kI8Rows * kI8Chunk, &maps.a, (c0 + it) * kI8Chunk, blockIdx.y * BN, &full[s]);
            }
            for (int j = max(0, it - C::kStages); j < it; j++)
                mbar_wait_err(&full[j % C::kStages], (j / C::kStages) & 1, err, kErrI8);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int it = 0;
            for (; it < nch; it++) {
                const int s = it % C::kStages;
                if (!wait(&full[s], (it / C::kStages) & 1)) break;
                tc_fence_after();
                const uint32_t st = smem_u32(sm + s * C::kStage);
                const uint64_t w = sw128_desc(st), a = sw128_desc(st + kI8Rows * kI8Chunk);
#pragma unroll
                for (int k = 0; k < kI8Chunk / 32; k++) i8_mma(tmem, w + 2 * k, a + 2 * k, i8_idesc(BN), it != 0 || k != 0);
                tc_commit(&empty[s]);
            }
            if (it == nch) tc_commit(&accf);
        }
    }
    int* const sums = reinterpret_cast<int*>(sm);  // [token][channel]; every product that read the stages is done
    const int q = warp & 3, j0 = blockIdx.x * kI8Rows, t0 = blockIdx.y * BN, live = min(BN, g.m - t0);
    if (warp >= 2) {
        constexpr int N = BN < 32 ? 16 : 32;
        float* const as = s_as[warp - 2];
        for (int c = lane; c < live; c += 32) as[c] = __ldg(g.as + t0 + c);
        __syncwarp();
        const bool ok = __all_sync(0xffffffffu, wait(&accf, 0));
        tc_fence_after();
        const uint32_t ta = tmem + ((uint32_t)(32 * q) << 16);
        if (ok && parts == 1) {
            i8_results<N>(g, ta, as, live, j0 + 32 * q + lane, g.C + (size_t)t0 * g.ldc + j0 + 32 * q + lane);
        } else if (ok) {
#pragma unroll 1
            for (int c = 0; c < live; c += N) {
                int v[N];
                if constexpr (N == 32)
                    i8_tmem_ld32(ta + c, v);
                else
                    i8_tmem_ld16(ta + c, v);
#pragma unroll
                for (int u = 0; u < N; u++) sums[(c + u) * kI8Rows + 32 * q + lane] = v[u];
            }
        }
    }
    if (parts > 1) {
        __syncwarp();
        i8_cluster_sync();
        if (warp >= 2) {
            // a warp takes a token of this CTA's share, a lane four channels, all parts' sums of it in flight
            const int j = j0 + 4 * lane, last = live * (z + 1) / parts;
            const bool wide = j + 3 < g.n && (((uintptr_t)g.C | (uintptr_t)(4 * (long long)g.ldc)) & 15) == 0;
            float ws[4], bias[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                ws[u] = j + u < g.n ? __ldg(g.ws + j + u) : 0.0f;
                bias[u] = g.bias && j + u < g.n ? __ldg(g.bias + j + u) : 0.0f;
            }
            for (int t = live * z / parts + q; t < last; t += 4) {
                const uint32_t at = smem_u32(sums + t * kI8Rows + 4 * lane);
                int4 v[8];
#pragma unroll
                for (int p = 0; p < 8; p++) {
                    v[p] = make_int4(0, 0, 0, 0);
                    if (p < parts) v[p] = i8_far(at, p);
                }
                int sum[4] = {0, 0, 0, 0};
#pragma unroll
                for (int p = 0; p < 8; p++) {
                    sum[0] += v[p].x;
                    sum[1] += v[p].y;
                    sum[2] += v[p].z;
                    sum[3] += v[p].w;
                }
                const float as = __ldg(g.as + t0 + t);
                float y[4];
#pragma unroll
                for (int u = 0; u < 4; u++) y[u] = i8_out(sum[u], as, ws[u], g.bias != nullptr, bias[u]);
                float* to = g.C + (size_t)(t0 + t) * g.ldc + j;
                if (wide)
                    *reinterpret_cast<float4*>(to) = make_float4(y[0], y[1], y[2], y[3]);
                else
#pragma unroll
                    for (int u = 0; u < 4; u++)
                        if (j + u < g.n) to[u] = y[u];
            }
        }
        __syncwarp();
        i8_cluster_sync();  // no CTA's memory goes while another one reads it
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, C::kCols);
    }
}

// Map of an array [rows][k] of bytes, boxes of 128 bytes of `box` rows.
int i8_map(CUtensorMap* m, const int8_t* base, int rows, int k, int ld, int box) {
    void* fn = nullptr;
    if (int e = tensor_map_encoder(&fn)) return e;
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
    const cuuint32_t boxes[2] = {kI8Chunk, (cuuint32_t)box}, step[2] = {1, 1};
    const CUresult r = reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(fn)(
        m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(base), dims, strides, boxes, step,
        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return cuda_fail(cudaErrorInvalidValue, "cuTensorMapEncodeTiled");
    return JYC_OK;
}

template <class Kernel>
int i8_start(Kernel kernel, const I8Gemm& g, const I8Maps& maps, dim3 grid, dim3 cluster, int threads, int smem, cudaStream_t s) {
    if (int e = max_dynamic_smem(reinterpret_cast<const void*>(kernel), smem)) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster.x;
    at[1].val.clusterDim.y = cluster.y;
    at[1].val.clusterDim.z = cluster.z;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    JYC_CUDA(cudaLaunchKernelEx(&cfg, kernel, g, maps, device_error_word()));
    JYC_LAUNCHED();
    return JYC_OK;
}

template <int BN>
int i8_few(const I8Gemm& g, I8Maps maps, int sms, cudaStream_t s) {
    if (int e = i8_map(&maps.a, g.A, g.m, g.k, g.lda, BN)) return e;
    const long long tiles = (long long)((g.n + kI8Rows - 1) / kI8Rows) * ((g.m + BN - 1) / BN);
    const int chunks = (g.k + kI8Chunk - 1) / kI8Chunk;
    // parts of K where the tiles leave many SMs idle, two CTAs on each at most (behind a flushed L2, the launch among them:
    // 128 tokens of 4096 x 4096, 32 tiles, 23 us in one part, 17 in four, 19 in eight; 48 tokens of 14336 x 4096, 112 tiles,
    // 26 us in one or two, 30 in four); more of them for long rows only (one token of 4096 x 14336 23 us in four, 22 in
    // eight; of 4096 x 4096 13.2 and 13.4)
    const int most = chunks >= 64 ? 8 : 4;
    int parts = 1;
    while (parts < most && tiles * 5 < 3 * sms && tiles * parts <= sms && chunks >= 4 * parts) parts *= 2;
    return i8_start(i8_few_kernel<BN>, g, maps, dim3((g.n + kI8Rows - 1) / kI8Rows, (g.m + BN - 1) / BN, parts),
                    dim3(1, 1, parts), kI8Threads, I8Few<BN>::kSmem, s);
}

}  // namespace

int launch_quantize_rows(const float* x, int ldx, int rows, int k, int8_t* q, int ldq, float* scale, cudaStream_t s) {
    const bool wide = aligned16(x, ldx) && ((uintptr_t)q & 3) == 0 && (ldq & 3) == 0;
    const int quads = (k + 4 * kQrThreads - 1) / (4 * kQrThreads);
    const auto kernel = !wide || quads > 16 ? quantize_rows_kernel<0>
                        : quads <= 1        ? quantize_rows_kernel<1>
                        : quads <= 4        ? quantize_rows_kernel<4>
                                            : quantize_rows_kernel<16>;
    return launch_follow(kernel, dim3(rows), kQrThreads, 0, s, x, ldx, k, q, ldq, scale);
}

int launch_i8_gemm(const I8Gemm& all, cudaStream_t s) {
    const int sms = sm_count();
    if (sms == 0) return cuda_fail(cudaErrorNoDevice, "matmul_i8: device query");
    I8Gemm g = all;
    I8Maps maps{};
    if (int e = i8_map(&maps.w, g.W, g.n, g.k, g.ldw, kI8Rows)) return e;
    const long long tiles = (long long)((g.n + 2 * kI8Rows - 1) / (2 * kI8Rows)) * ((g.m + kI8PairTokens - 1) / kI8PairTokens);
    // the pairs' tiles for a quarter of the SMs or more (129 tokens of 14336 x 4096 27 us, 29 in few tiles; 256 of 4096 x
    // 4096 22 against 18)
    if (g.m > 128 && g.n > kI8Rows && tiles * 4 > sms) {
        if (int e = i8_map(&maps.a, g.A, g.m, g.k, g.lda, kI8PairTokens / 2)) return e;
        return i8_start(i8_pair_kernel, g, maps, dim3(2 * (unsigned)std::min<long long>(tiles, sms / 2)), dim3(2, 1, 1),
                        kI8PairThreads, kI8PairSmem, s);
    }
    if (g.m <= 16) return i8_few<16>(g, maps, sms, s);
    if (g.m <= 32) return i8_few<32>(g, maps, sms, s);
    if (g.m <= 64) return i8_few<64>(g, maps, sms, s);
    const int most = 65535 * 128;  // token tiles of a launch
    for (int r0 = 0; r0 < all.m; r0 += most) {
        g.A = all.A + (size_t)r0 * all.lda;
        g.as = all.as + r0;
        g.C = all.C + (size_t)r0 * all.ldc;
        g.m = std::min(most, all.m - r0);
        if (int e = i8_few<128>(g, maps, sms, s)) return e;
        if (all.m - r0 <= most) break;
    }
    return JYC_OK;
}

}  // namespace jyc
