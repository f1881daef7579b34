// rope.cuh — rotary positions of rows in either pair layout, over a part of the head (rope.cu, and as
// rows are appended to or attend over the 4-bit pages, paged4.cu).
#pragma once
#include "paged.cuh"

namespace jyc {

struct RopeView {
    const float* cos_t;  // nullptr: rows arrive turned
    const float* sin_t;
    int len;   // rows of the tables
    int half;  // pairs of a head
    bool halves;
};

// One pair turned: rope_pos's rounding, one product rounded, one fused sum.
__device__ __forceinline__ void turn_pair(float a, float b, float c, float s, float& r0, float& r1) {
    r0 = __fmaf_rn(a, c, -__fmul_rn(b, s));
    r1 = __fmaf_rn(a, s, __fmul_rn(b, c));
}

// Dims d0 .. d0 + 3 of a head at x (hd floats), turned by row `pos` of the tables. vec: heads and table rows lie on
// 16 bytes and the rotated part ends, and its halves meet, on a multiple of 4 dims.
__device__ __forceinline__ float4 turned4(const float* x, int d0, const RopeView& r, int pos, bool vec) {
    const int rot = 2 * r.half;
    const float* ct = r.cos_t + (size_t)pos * r.half;
    const float* st = r.sin_t + (size_t)pos * r.half;
    float4 y;
    if (vec) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(x + d0));
        if (d0 >= rot) return v;
        if (r.halves) {
            const bool first = d0 < r.half;
            const int i = first ? d0 : d0 - r.half;
            const float4 w = __ldg(reinterpret_cast<const float4*>(x + (first ? d0 + r.half : i)));
            const float4 c = __ldg(reinterpret_cast<const float4*>(ct + i)), s = __ldg(reinterpret_cast<const float4*>(st + i));
            const float4 a = first ? v : w, b = first ? w : v;
            float4 r0, r1;
            turn_pair(a.x, b.x, c.x, s.x, r0.x, r1.x);
            turn_pair(a.y, b.y, c.y, s.y, r0.y, r1.y);
            turn_pair(a.z, b.z, c.z, s.z, r0.z, r1.z);
            turn_pair(a.w, b.w, c.w, s.w, r0.w, r1.w);
            return first ? r0 : r1;
        }
        const float2 c = __ldg(reinterpret_cast<const float2*>(ct + d0 / 2)), s = __ldg(reinterpret_cast<const float2*>(st + d0 / 2));
        turn_pair(v.x, v.y, c.x, s.x, y.x, y.y);
        turn_pair(v.z, v.w, c.y, s.y, y.z, y.w);
        return y;
    }
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int d = d0 + i;
        o[i] = __ldg(x + d);
        if (d >= rot) continue;
        const int j = r.halves ? (d < r.half ? d : d - r.half) : d >> 1;
        const bool first = r.halves ? d < r.half : !(d & 1);
        const float other = __ldg(x + (r.halves ? (first ? d + r.half : j) : d ^ 1));
        float r0, r1;
        turn_pair(first ? o[i] : other, first ? other : o[i], __ldg(ct + j), __ldg(st + j), r0, r1);
        o[i] = first ? r0 : r1;
    }
    return make_float4(o[0], o[1], o[2], o[3]);
}
// Whether turned4 may take its wide form: x's rows and heads, and the tables.
inline bool rope_wide(const RopeView& r) {
    return (((uintptr_t)r.cos_t | (uintptr_t)r.sin_t) & 15) == 0 && r.half % (r.halves ? 4 : 2) == 0;
}

int launch_rope_rows(const float* X, int ldx, float* Y, int ldy, int rows, int H, int hd, const int* row_pos,
                     const RopeView& r, cudaStream_t s);

}  // namespace jyc
