// paged4.cuh — K/V cache in 4-bit groups of 32 dims, in pages: append, read back, attention of one new
// token per sequence that leaves its weights, eviction by them (paged4.cu).
#pragma once
#include "paged.cuh"
#include "rope.cuh"

namespace jyc {

// Where a position of a sequence lives, as PagedKV for jyc_kv_pages_q4.
struct PagedKV4 {
    jyc_kv_pages_q4 p;
    const int* table;
    int table_stride;
    int num_seqs;
    FastDiv by_page;
    int* err;  // the paged error word
};

int launch_paged4_append(const float* K, const float* V, int ld, int rows, int KV, int hd, const int* row_seq,
                         const int* row_pos, const int* rope_pos, const PagedKV4& kv, const RopeView& rope,
                         cudaStream_t s);
int launch_paged4_read(float* K, float* V, int ld, int rows, int KV, int hd, const int* row_seq, const int* row_pos,
                       const PagedKV4& kv, cudaStream_t s);

struct PagedAttn4 {
    const float* Q;
    int ldq;
    float* out;
    int ldo;
    int H, KV, hd;
    const int* lens;
    const int* rope_pos;  // nullptr: lens - 1
    PagedKV4 kv;
    RopeView rope;
    float scale;  // 1/sqrtf(hd)
};
// capacity: positions of a sequence where the weights are gathered, else 0. 0 bytes: no device.
size_t paged4_attention_workspace(int seqs, int H, int KV, int hd, int capacity);
int launch_paged4_attention(const PagedAttn4& a, void* work, cudaStream_t s);

struct PagedEvict4 {
    const int* lens;
    int budget, recent;
    int KV, hd;
    PagedKV4 kv;
    const int* new_table;
    int new_stride;
    int* new_lens;
    int* kept;
};
int launch_paged4_evict(const PagedEvict4& e, cudaStream_t s);

}  // namespace jyc
