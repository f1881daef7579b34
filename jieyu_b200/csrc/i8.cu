// i8.cu — C = (A W^T) * (a_scale w_scale) + bias over 8-bit integers with 32-bit sums, and the rows of
// fp32 activations in 8 bits that go into it (kv_pack_q8's rule over a whole row,
// libs/model_libs/attention/attention_q8.h:24-35).
#include "i8.cuh"

#include <algorithm>

namespace jyc {

namespace {

constexpr int kQrThreads = 256;

// A CTA quantises one row: its maximum, then its values, read again.
__global__ void __launch_bounds__(kQrThreads) quantize_rows_kernel(const float* x, int ldx, int k, int8_t* q, int ldq,
                                                                   float* scale) {
    __shared__ float s_max[kQrThreads / 32];
    const int tid = threadIdx.x;
    const float* row = x + (size_t)blockIdx.x * ldx;
    int8_t* to = q + (size_t)blockIdx.x * ldq;
    float amax = 0.0f;
    for (int i = tid; i < k; i += kQrThreads) amax = fmaxf(amax, fabsf(__ldg(row + i)));
    amax = warp_max(amax);
    if ((tid & 31) == 0) s_max[tid >> 5] = amax;
    __syncthreads();
    for (int w = 0; w < kQrThreads / 32; w++) amax = fmaxf(amax, s_max[w]);
    const float inv = q8_inv(amax);
    if (tid == 0) scale[blockIdx.x] = q8_scale(amax);
    for (int i = tid; i < k; i += kQrThreads) to[i] = (int8_t)q8_round(__ldg(row + i), inv);
}

// Sum, scales and bias: one rounding each.
__device__ __forceinline__ float i8_out(int sum, float as, float ws, const float* bias, int j) {
    const float v = __fmul_rn(__int2float_rn(sum), __fmul_rn(as, ws));
    return bias ? __fadd_rn(v, __ldg(bias + j)) : v;
}

// A warp computes one output channel for up to 8 rows: lanes along k.
__global__ void __launch_bounds__(256) i8_simple_kernel(I8Gemm g) {
    const int j = blockIdx.x * 8 + (threadIdx.x >> 5), i0 = blockIdx.y * 8, lane = threadIdx.x & 31;
    if (j >= g.n) return;
    int acc[8] = {};
    for (int k = lane; k < g.k; k += 32) {
        const int w = g.W[(size_t)j * g.ldw + k];
        for (int r = 0; r < 8; r++)
            if (i0 + r < g.m) acc[r] += w * g.A[(size_t)(i0 + r) * g.lda + k];
    }
    for (int r = 0; r < 8; r++) {
        int v = acc[r];
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0 && i0 + r < g.m)
            g.C[(size_t)(i0 + r) * g.ldc + j] = i8_out(v, __ldg(g.as + i0 + r), __ldg(g.ws + j), g.bias, j);
    }
}

}  // namespace

int launch_quantize_rows(const float* x, int ldx, int rows, int k, int8_t* q, int ldq, float* scale, cudaStream_t s) {
    quantize_rows_kernel<<<rows, kQrThreads, 0, s>>>(x, ldx, k, q, ldq, scale);
    JYC_LAUNCHED();
    return JYC_OK;
}

int launch_i8_gemm(const I8Gemm& a, cudaStream_t s) {
    const int most = 8 * 65535;
    for (int r0 = 0; r0 < a.m; r0 += most) {
        I8Gemm g = a;
        g.A += (size_t)r0 * a.lda;
        g.as += r0;
        g.C += (size_t)r0 * a.ldc;
        g.m = std::min(most, a.m - r0);
        i8_simple_kernel<<<dim3((g.n + 7) / 8, (g.m + 7) / 8), 256, 0, s>>>(g);
        JYC_LAUNCHED();
        if (a.m - r0 <= most) break;
    }
    return JYC_OK;
}

}  // namespace jyc
