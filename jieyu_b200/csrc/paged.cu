// paged.cu — int8 K/V cache in pages: rows are quantised as they are written
// (kv_pack_q8's rule, libs/model_libs/attention/attention_q8.h:20-37), read
// back as fp32, and attended over by one new token per sequence (the score,
// softmax and P.V of attention_q8.h:38-184).
#include "paged.cuh"

#include <algorithm>

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

// CTA = (query head, sequence), 8 warps; warp w takes positions w, w + 8, ...
// with its own online softmax: one position at a time, a lane holds up to 8
// dims. The warps' (m, l, o) are joined at the end.
constexpr int kSimpleWarps = 8;

__global__ void __launch_bounds__(kSimpleWarps * 32) paged_attention_kernel(PagedAttn a) {
    __shared__ float s_m[kSimpleWarps], s_l[kSimpleWarps], s_o[kSimpleWarps][256];
    const int h = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kvh = h / (a.H / a.KV), hd = a.hd, half = hd >> 1, nq = hd >> 2;
    int len = a.lens[b];
    const long long cap = (long long)a.kv.table_stride * a.kv.p.page_size;
    if (len > cap) {
        paged_flag(kPagedErrPos);
        len = (int)cap;
    }
    float* out = a.out + (size_t)b * a.ldo + (size_t)h * hd;
    if (len > 0 && a.rope.cos_t && len > a.rope.len) {
        paged_flag(kPagedErrRope);
        len = 0;
    }
    if (len <= 0) {
        for (int e = threadIdx.x; e < hd; e += blockDim.x) out[e] = 0.0f;
        return;
    }
    float4 x[2];
    int slot4[2];
    float amax = 0.0f;
    for (int t = 0; t < 2; t++) {
        const int qd = lane + 32 * t;
        slot4[t] = qd;
        x[t] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (qd >= nq) continue;
        x[t] = load4(a.Q + (size_t)b * a.ldq + (size_t)h * hd + 4 * qd, false);
        if (a.rope.cos_t) {
            x[t] = rotate4(x[t], a.rope.cos_t + (size_t)(len - 1) * half, a.rope.sin_t + (size_t)(len - 1) * half, qd);
            slot4[t] = rope_slot(2 * qd, half) >> 1;
        }
        amax = fmaxf(amax, amax4(x[t]));
    }
    amax = warp_max(amax);
    const float inv = q8_inv(amax), qs = q8_scale(amax);
    const uint32_t q[2] = {pack4(x[0], inv), pack4(x[1], inv)};
    float m = -INFINITY, l = 0.0f, o[2][4] = {};
    for (int j = warp; j < len; j += kSimpleWarps) {
        const int page = paged_page(a.kv, b, j);
        if (page < 0) continue;
        const int slot = j % a.kv.p.page_size;
        const uint32_t* kr = reinterpret_cast<const uint32_t*>(a.kv.p.k + paged_off(a.kv, page, slot, kvh));
        const uint32_t* vr = reinterpret_cast<const uint32_t*>(a.kv.p.v + paged_off(a.kv, page, slot, kvh));
        int dot = 0;
        for (int t = 0; t < 2; t++)
            if (lane + 32 * t < nq) dot = __dp4a((int)q[t], (int)kr[slot4[t]], dot);
        for (int i = 16; i > 0; i >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, i);
        const size_t so = paged_soff(a.kv, page, slot, kvh);
        const float sc = __fmul_rn((float)dot, __fmul_rn(__fmul_rn(a.kv.p.ks[so], qs), a.scale));
        const float mn = fmaxf(m, sc);
        const float al = m == -INFINITY ? 0.0f : expf(m - mn), e = expf(sc - mn), w = e * a.kv.p.vs[so];
        m = mn;
        l = l * al + e;
        for (int t = 0; t < 2; t++) {
            float f[4] = {};
            if (lane + 32 * t < nq) u8x4_to_f32(vr[lane + 32 * t] ^ 0x80808080u, f);
            for (int i = 0; i < 4; i++) o[t][i] = __fmaf_rn(w, f[i], o[t][i] * al);
        }
    }
    if (lane == 0) {
        s_m[warp] = m;
        s_l[warp] = l;
    }
    for (int t = 0; t < 2; t++)
        if (lane + 32 * t < nq)
            for (int i = 0; i < 4; i++) s_o[warp][4 * (lane + 32 * t) + i] = o[t][i];
    __syncthreads();
    float M = -INFINITY, L = 0.0f;
    for (int w = 0; w < kSimpleWarps; w++) M = fmaxf(M, s_m[w]);
    for (int e = threadIdx.x; e < hd; e += blockDim.x) {
        float O = 0.0f;
        L = 0.0f;
        for (int w = 0; w < kSimpleWarps; w++) {
            if (s_m[w] == -INFINITY) continue;
            const float wgt = expf(s_m[w] - M);
            L = __fmaf_rn(wgt, s_l[w], L);
            O = __fmaf_rn(wgt, s_o[w][e], O);
        }
        out[e] = M == -INFINITY ? 0.0f : O / L;
    }
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

size_t paged_attention_workspace(int, int, int, int) { return 16; }

int launch_paged_attention(const PagedAttn& a, void*, cudaStream_t s) {
    paged_attention_kernel<<<dim3(a.H, a.kv.num_seqs), kSimpleWarps * 32, 0, s>>>(a);
    JYC_LAUNCHED();
    return JYC_OK;
}

}  // namespace jyc
