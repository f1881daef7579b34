// paged.cuh — int8 K/V cache in pages shared by many sequences: append, read
// back, attention of one new token per sequence (paged.cu), and the batched
// token pick (pick.cu).
#pragma once
#include "common.cuh"

namespace jyc {

// n / d for 0 <= n < 2^31 by a multiplication: with 2^(s-1) < d <= 2^s and m = ceil(2^(31+s) / d) < 2^32, m d -
// 2^(31+s) < d <= 2^s, so n m / 2^(31+s) is above n / d by less than n 2^-31 / d < 1 / d.
struct FastDiv {
    uint32_t m;
    int s;
    __device__ __forceinline__ int operator()(int n) const { return (int)(((unsigned long long)(uint32_t)n * m) >> s); }
};
inline FastDiv fast_div(int d) {
    int s = 0;
    while ((1LL << s) < d) s++;
    return FastDiv{(uint32_t)(((1ULL << (31 + s)) + (unsigned)d - 1) / (unsigned)d), 31 + s};
}

// Where a position of a sequence lives: page id = table[seq * table_stride +
// pos / page_size], then the strides of jyc_kv_pages.
struct PagedKV {
    jyc_kv_pages p;
    const int* table;
    int table_stride;  // table entries per sequence
    int num_seqs;
    FastDiv by_page;   // position / page_size
};

struct PagedRope {
    const float* cos_t;  // nullptr: rows arrive rotated
    const float* sin_t;
    int len;             // rows of the tables
};

// bits of the paged error word
constexpr int kPagedErrPos = 1;   // sequence or position out of range
constexpr int kPagedErrPage = 2;  // page id out of range
constexpr int kPagedErrRope = 4;  // position behind the RoPE tables
constexpr int kPagedErrWait = 8;  // a copy's bounded wait gave up

int* paged_error_word();
// Clears these bits, and no other that a call sets meanwhile; they are clear on return.
int paged_error_clear(int bits);
// Rows of ld floats at p lie on 16 bytes.
inline bool aligned16(const void* p, int ld) { return ((uintptr_t)p & 15) == 0 && (ld & 3) == 0; }
// SMs of the current device (0: no device).
int sm_count();
// The kernel's limit of dynamic shared memory on the current device, set once for each.
int max_dynamic_smem(const void* kernel, int bytes);

int launch_paged_append(const float* K, const float* V, int ld, int rows, int KV, int hd, const int* row_seq,
                        const int* row_pos, const PagedKV& kv, const PagedRope& rope, cudaStream_t s);
int launch_paged_read(float* K, float* V, int ld, int rows, int KV, int hd, const int* row_seq, const int* row_pos,
                      const PagedKV& kv, cudaStream_t s);

struct PagedAttn {
    const float* Q;
    int ldq;
    float* out;
    int ldo;
    int H, KV, hd;
    const int* lens;
    PagedKV kv;
    PagedRope rope;
    float scale;  // 1/sqrtf(hd)
};
size_t paged_attention_workspace(int H, int KV, int hd);
int launch_paged_attention(const PagedAttn& a, void* work, cudaStream_t s);

struct PickArgs {
    const float* logits;
    int ld, rows, V;
    const float* temperature;  // any of these arrays may be null (see jyc_sample_batch)
    const int* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
    int* ids;
    float* probs;  // may be null
};
constexpr int kPickMaxVocab = 1 << 20;  // weights are 2^42 fixed point: 2^20 of them fit 64 bits
int launch_pick(const PickArgs& a, cudaStream_t s);

}  // namespace jyc
