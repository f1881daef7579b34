// rope.cu — rotary positions of rows (rope_pos's rotation, libs/model_libs/rope/rope.h:108-110, for any row
// positions, both pair layouts and a part of the head).
#include "rope.cuh"

#include <algorithm>

namespace jyc {

namespace {

constexpr int kRopeThreads = 128;

// A thread turns one pair, or copies one dim behind the rotated part.
__global__ void __launch_bounds__(kRopeThreads) rope_rows_kernel(const float* X, int ldx, float* Y, int ldy, int H,
                                                                 int hd, const int* row_pos, RopeView r, int items,
                                                                 int chunks, int* err) {
    const int row = blockIdx.x / chunks, f = (blockIdx.x - row * chunks) * kRopeThreads + threadIdx.x;
    if (f >= H * items) return;
    const int head = f / items, i = f - head * items;
    const int pos = __ldg(row_pos + row);
    if (pos < 0) return;
    if (pos >= r.len) {
        atomicOr(err, kPagedErrRope);
        return;
    }
    const float* x = X + (size_t)row * ldx + (size_t)head * hd;
    float* y = Y + (size_t)row * ldy + (size_t)head * hd;
    if (i >= r.half) {
        y[i + r.half] = x[i + r.half];
        return;
    }
    const int a = r.halves ? i : 2 * i, b = r.halves ? i + r.half : 2 * i + 1;
    float r0, r1;
    turn_pair(x[a], x[b], r.cos_t[(size_t)pos * r.half + i], r.sin_t[(size_t)pos * r.half + i], r0, r1);
    y[a] = r0;
    y[b] = r1;
}

}  // namespace

int launch_rope_rows(const float* X, int ldx, float* Y, int ldy, int rows, int H, int hd, const int* row_pos,
                     const RopeView& r, cudaStream_t s) {
    int* err = paged_error_word();
    if (!err) return cuda_fail(cudaErrorNoDevice, "rope_rows: error word");
    const int items = hd - r.half, chunks = (int)(((long long)H * items + kRopeThreads - 1) / kRopeThreads);
    const int most = std::max(1, 0x7fffffff / chunks);
    for (int r0 = 0; r0 < rows; r0 += most) {
        const int n = std::min(most, rows - r0);
        rope_rows_kernel<<<(unsigned)n * chunks, kRopeThreads, 0, s>>>(X + (size_t)r0 * ldx, ldx, Y + (size_t)r0 * ldy,
                                                                       ldy, H, hd, row_pos + r0, r, items, chunks, err);
        JYC_LAUNCHED();
        if (rows - r0 <= most) break;
    }
    return JYC_OK;
}

}  // namespace jyc
