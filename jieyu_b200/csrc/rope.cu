// rope.cu — rotary positions of rows (rope_pos's rotation, libs/model_libs/rope/rope.h:108-110, for any row
// positions, both pair layouts and a part of the head).
#include "rope.cuh"
#include "follow.cuh"
#include "ptx.cuh"

#include <algorithm>

namespace jyc {

namespace {

constexpr int kRopeThreads = 128;
constexpr int kRopeHeads = 4;  // heads of a thread

// Bound by memory: 8 bytes a value. A thread keeps one item of a head (two quads that turn together, or one quad: two
// pairs of neighbours, or four dims that stay) in up to kRopeHeads heads of a row, all of whose loads are in flight
// at once; its table entries are read once for all of them. Neighbouring threads hold neighbouring items, then
// heads. It reads all that it turns before it writes, so Y may be X. Measured: 16384 rows of 40 x 128, half of each head
// turned, 99 us, 6.8 TB/s (293 us with a pair or a dim a thread); 64 rows 4 us, most of the call's 8 its launch.
template <bool HALVES>
__global__ void __launch_bounds__(kRopeThreads) rope_rows_kernel(const float* X, int ldx, float* Y, int ldy, int H,
                                                                 int hd, const int* row_pos, RopeView r, int items,
                                                                 int side, int steps, int chunks, int* err) {
    griddep_wait();
    const int row = blockIdx.x / chunks, chunk = blockIdx.x - row * chunks, at = threadIdx.x / items;
    if (at >= side) return;
    const int i = threadIdx.x - at * items, rot = 2 * r.half, turning = HALVES ? r.half / 4 : rot / 4;
    const int pos = __ldg(row_pos + row);
    if (pos < 0) return;
    if (pos >= r.len) {
        if (i == 0) atomicOr(err, kPagedErrRope);
        return;
    }
    const bool turns = i < turning;
    const int d0 = turns ? 4 * i : rot + 4 * (i - turning), d1 = HALVES && turns ? d0 + r.half : d0;
    const int h0 = chunk * steps * side + at;
    const float* x = X + (size_t)row * ldx + (size_t)h0 * hd;
    float* y = Y + (size_t)row * ldy + (size_t)h0 * hd;
    float4 a[kRopeHeads], b[kRopeHeads], c, s;
    c = s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (turns) {
        const float* ct = r.cos_t + (size_t)pos * r.half;
        const float* st = r.sin_t + (size_t)pos * r.half;
        if (HALVES) {
            c = __ldg(reinterpret_cast<const float4*>(ct + d0));
            s = __ldg(reinterpret_cast<const float4*>(st + d0));
        } else {
            const float2 c2 = __ldg(reinterpret_cast<const float2*>(ct + d0 / 2));
            const float2 s2 = __ldg(reinterpret_cast<const float2*>(st + d0 / 2));
            c.x = c2.x; c.y = c2.y; s.x = s2.x; s.y = s2.y;
        }
    }
#pragma unroll
    for (int u = 0; u < kRopeHeads; u++)
        if (u < steps && h0 + u * side < H) {
            a[u] = *reinterpret_cast<const float4*>(x + (size_t)u * side * hd + d0);
            if (HALVES && turns) b[u] = *reinterpret_cast<const float4*>(x + (size_t)u * side * hd + d1);
        }
#pragma unroll
    for (int u = 0; u < kRopeHeads; u++)
        if (u < steps && h0 + u * side < H) {
            float* to = y + (size_t)u * side * hd;
            float4 v = a[u], w;
            if (turns && HALVES) {
                turn_pair(a[u].x, b[u].x, c.x, s.x, v.x, w.x);
                turn_pair(a[u].y, b[u].y, c.y, s.y, v.y, w.y);
                turn_pair(a[u].z, b[u].z, c.z, s.z, v.z, w.z);
                turn_pair(a[u].w, b[u].w, c.w, s.w, v.w, w.w);
                *reinterpret_cast<float4*>(to + d1) = w;
            } else if (turns) {
                turn_pair(a[u].x, a[u].y, c.x, s.x, v.x, v.y);
                turn_pair(a[u].z, a[u].w, c.y, s.y, v.z, v.w);
            }
            *reinterpret_cast<float4*>(to + d0) = v;
        }
}

// Shapes that do not lie on quads, which are rare: a thread turns one pair, or copies one dim behind the rotated part.
// (16384 rows of 40 x 128 that lie off 16 bytes, half of each head turned: 305 us, 102 where they lie on quads.)
__global__ void __launch_bounds__(kRopeThreads) rope_rows_odd_kernel(const float* X, int ldx, float* Y, int ldy, int H,
                                                                     int hd, const int* row_pos, RopeView r, int items,
                                                                     int chunks, int* err) {
    griddep_wait();
    const int row = blockIdx.x / chunks;
    const unsigned f = (blockIdx.x - row * chunks) * kRopeThreads + threadIdx.x;  // up to 127 behind H * items < 2^31
    if (f >= (unsigned)(H * items)) return;
    const int head = (int)(f / items), i = (int)(f - head * items);
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
    // quads: heads, table rows and the rotated part on 16 bytes, a head's items within a CTA
    const int quads = (r.halves ? r.half : 2 * r.half) / 4 + (hd - 2 * r.half) / 4;
    const bool wide = hd % 4 == 0 && aligned16(X, ldx) && aligned16(Y, ldy) && rope_wide(r) && quads <= kRopeThreads;
    const int items = wide ? quads : hd - r.half, side = wide ? kRopeThreads / items : 0;
    const int all = wide ? (H + side - 1) / side : 0;  // steps of a row
    const int chunks = wide ? (all + kRopeHeads - 1) / kRopeHeads
                            : (int)(((long long)H * items + kRopeThreads - 1) / kRopeThreads);
    const int steps = wide ? (all + chunks - 1) / chunks : 0, most = std::max(1, 0x7fffffff / chunks);
    for (int r0 = 0; r0 < rows; r0 += most) {
        const int n = std::min(most, rows - r0);
        const float* x = X + (size_t)r0 * ldx;
        float* y = Y + (size_t)r0 * ldy;
        const dim3 grid((unsigned)n * chunks);
        const auto kernel = r.halves ? rope_rows_kernel<true> : rope_rows_kernel<false>;
        if (int e = wide ? launch_follow(kernel, grid, kRopeThreads, 0, s, x, ldx, y, ldy, H, hd, row_pos + r0, r, items, side,
                                         steps, chunks, err)
                         : launch_follow(rope_rows_odd_kernel, grid, kRopeThreads, 0, s, x, ldx, y, ldy, H, hd, row_pos + r0, r,
                                         items, chunks, err))
            return e;
        if (rows - r0 <= most) break;
    }
    return JYC_OK;
}

}  // namespace jyc
