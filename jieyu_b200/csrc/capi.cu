// capi.cu — operator-level C ABI over device pointers (one entry per reference
// operator; see include/jieyu_b200.h for the reference function each replaces).
#include <algorithm>
#include <cmath>
#include <mutex>
#include <vector>

#include "i8.cuh"
#include "kernels.cuh"
#include "mega.cuh"
#include "paged.cuh"
#include "paged4.cuh"
#include "rope.cuh"
#include "tcgemm.cuh"
#include "skinny.cuh"

using namespace jyc;

namespace {

#define TRY(x)                          \
    do {                                \
        int _r = (x);                   \
        if (_r != JYC_OK) return _r;    \
    } while (0)

inline cudaStream_t S(void* s) { return static_cast<cudaStream_t>(s); }

// Stream-ordered scratch for one op call (freed in stream order).
struct Scratch {
    cudaStream_t s;
    std::vector<void*> ptrs;
    explicit Scratch(cudaStream_t st) : s(st) {}
    template <class T>
    int get(T** p, size_t count) {
        void* q = nullptr;
        cudaError_t e = cudaMallocAsync(&q, std::max<size_t>(count, 1) * sizeof(T), s);
        if (e != cudaSuccess) return cuda_fail(e, "cudaMallocAsync");
        ptrs.push_back(q);
        *p = static_cast<T*>(q);
        return JYC_OK;
    }
    ~Scratch() {
        for (void* q : ptrs) cudaFreeAsync(q, s);
    }
};

}  // namespace

extern "C" {

JYC_API int jyc_q8_repack(const void* blocks, int n, int k, uint8_t* qs, uint16_t* d, void* stream) {
    clear_error();
    if (!blocks || !qs || !d) return arg_error("q8_repack: null pointer");
    return launch_q8_repack(blocks, n, k, qs, d, 0, 1, S(stream));
}

JYC_API int jyc_matmul_q8(const float* A, const uint8_t* qs, const uint16_t* d, float* C, int m,
                          int n, int k, void* stream) {
    clear_error();
    if (!A || !qs || !d || !C) return arg_error("matmul_q8: null pointer");
    if (m <= 0 || n <= 0 || k <= 0 || k % 32) return arg_error("matmul_q8: need m,n > 0 and k % 32 == 0");
    if (m >= kTcMinRows) {
        // a real contraction: tcgen05 tiles of 128 weight rows x up to 128 rows of A
        cudaStream_t s = S(stream);
        int N = 0, splits = 1;
        tc_plan(n, k, m, kTcMaxSplits, &N, &splits);
        Scratch sc(s);
        __half* xs = nullptr;
        int* xe = nullptr;
        TRY(sc.get(&xs, tc_split_halves(m, N, k)));
        TRY(sc.get(&xe, (size_t)tc_padded_tokens(m, N)));
        uint8_t* rexp = nullptr;
        TRY(sc.get(&rexp, (size_t)n));
        TRY(launch_tc_rowexp(d, n, k, rexp, s));
        TRY(launch_tc_split(A, k, m, k, nullptr, 0.0f, N, xs, xe, s));
        TcGemm g{};
        g.qs = qs; g.d = d; g.rexp = rexp; g.n = n; g.k = k; g.xs = xs; g.xe = xe; g.T = m; g.N = N;
        g.y = C; g.ldy = n; g.err = device_error_word();
        g.splits = splits;
        if (g.splits > 1) {
            const size_t tiles = (size_t)((n + kTcRows - 1) / kTcRows) * ((m + N - 1) / N);
            TRY(sc.get(&g.part, (size_t)g.splits * m * n));
            TRY(sc.get(&g.cnt, tiles));
            JYC_CUDA(cudaMemsetAsync(g.cnt, 0, tiles * sizeof(unsigned int), s));
        }
        return launch_tc_gemm(g, TC_STORE, s);
    }
    if (m > 1 && ((uintptr_t)A & 15) == 0 && ((uintptr_t)qs & 15) == 0) {
        // a few rows: activations in registers, weights streamed once per 8 rows
        cudaStream_t s = S(stream);
        Scratch sc(s);
        SkinnyWork w{};
        const size_t cnt = skinny_counters(n);
        TRY(sc.get(&w.part, skinny_part_floats(n, k)));
        TRY(sc.get(&w.cnt, cnt));
        JYC_CUDA(cudaMemsetAsync(w.cnt, 0, cnt * sizeof(unsigned int), s));
        for (int r0 = 0; r0 < m; r0 += kSkMaxRows) {
            SkinnyGemm g{};
            g.x = A + (size_t)r0 * k; g.ldx = k; g.m = std::min(kSkMaxRows, m - r0); g.n = n; g.k = k;
            g.qs = qs; g.d = d; g.y = C + (size_t)r0 * n; g.ldy = n;
            TRY(launch_skinny(g, EPI_STORE, w, s));
        }
        return JYC_OK;
    }
    for (int r0 = 0; r0 < m; r0 += 8) {
        GemvArgs g{};
        g.x = A + (size_t)r0 * k; g.ldx = k; g.m = std::min(8, m - r0); g.n = n; g.k = k;
        g.qs = qs; g.d = d; g.y = C + (size_t)r0 * n; g.ldy = n;
        TRY(launch_gemv(g, W_Q8, EPI_STORE, S(stream)));
    }
    return JYC_OK;
}

JYC_API int jyc_matmul_qk(const float* A, const void* blocks, float* C, int m, int n, int k, int qtype,
                          void* stream) {
    clear_error();
    if (!A || !blocks || !C) return arg_error("matmul_qk: null pointer");
    return launch_kquant_matmul(A, m, n, k, static_cast<const uint8_t*>(blocks), qtype, C, S(stream));
}

JYC_API int jyc_f32_transpose(const float* B, float* Bt, int k, int n, void* stream) {
    clear_error();
    if (!B || !Bt) return arg_error("f32_transpose: null pointer");
    return launch_transpose(B, Bt, k, n, 0, 1, S(stream));
}

JYC_API int jyc_matmul_f32(const float* A, const float* Bt, float* C, int m, int n, int k,
                           void* stream) {
    clear_error();
    if (!A || !Bt || !C) return arg_error("matmul_f32: null pointer");
    if (m <= 0 || n <= 0 || k <= 0) return arg_error("matmul_f32: empty shape");
    if (k % 8 == 0 && m <= 8) {
        GemvArgs g{};
        g.x = A; g.ldx = k; g.m = m; g.n = n; g.k = k; g.wt = Bt; g.y = C; g.ldy = n;
        return launch_gemv(g, W_F32, EPI_STORE, S(stream));
    }
    return launch_matmul_f32_generic(A, Bt, C, m, n, k, S(stream));
}

JYC_API int jyc_f16_transpose(const uint16_t* B, uint16_t* Bt, int k, int n, void* stream) {
    clear_error();
    if (!B || !Bt) return arg_error("f16_transpose: null pointer");
    return launch_transpose_h(B, Bt, k, n, 0, 1, S(stream));
}

JYC_API int jyc_matmul_f16(const float* A, const uint16_t* Bt, float* C, int m, int n, int k,
                           void* stream) {
    clear_error();
    if (!A || !Bt || !C) return arg_error("matmul_f16: null pointer");
    if (m <= 0 || n <= 0 || k <= 0) return arg_error("matmul_f16: empty shape");
    if (k % 8 == 0 && m <= 8) {
        GemvArgs g{};
        g.x = A; g.ldx = k; g.m = m; g.n = n; g.k = k; g.wh = Bt; g.y = C; g.ldy = n;
        return launch_gemv(g, W_F16, EPI_STORE, S(stream));
    }
    return launch_matmul_f16_generic(A, Bt, C, m, n, k, S(stream));
}

JYC_API int jyc_rmsnorm(const float* x, float* y, const float* w, int rows, int n, float eps,
                        void* stream) {
    clear_error();
    if (!x || !y || !w) return arg_error("rmsnorm: null pointer");
    return launch_rmsnorm(x, y, w, rows, n, eps, S(stream));
}

JYC_API int jyc_rope_pos(float* q, int seq, int start_pos, int num_heads, int head_dim,
                         const float* cos_table, const float* sin_table, void* stream) {
    clear_error();
    if (!q || !cos_table || !sin_table) return arg_error("rope_pos: null pointer");
    if (seq < 0 || start_pos < 0 || num_heads <= 0 || head_dim <= 0) return arg_error("rope_pos: bad shape");
    return launch_rope(q, seq, start_pos, num_heads, head_dim, cos_table, sin_table, S(stream));
}

JYC_API int jyc_kv_pack_q8(const float* src, int8_t* dst, float* scale, int heads, int head_dim,
                           int n, void* stream) {
    clear_error();
    if (!src || !dst || !scale) return arg_error("kv_pack_q8: null pointer");
    if (heads <= 0 || head_dim <= 0 || n < 0) return arg_error("kv_pack_q8: bad shape");
    return launch_kv_pack(src, dst, scale, heads, head_dim, n, S(stream));
}

JYC_API int jyc_attention_q8(const float* Q, const float* K, const float* V, float* out, int seq,
                             int start_pos, int num_heads, int num_kv_heads, int head_dim,
                             int8_t* kc, float* ks, int8_t* vc, float* vs, int cap, void* stream) {
    clear_error();
    // argument checks of attention/x86/x86_classic.txt:2-8
    if (num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
        return arg_error("attention_q8: num_heads must be a multiple of num_kv_heads");
    if (seq <= 0) return arg_error("attention_q8: seq must be positive");
    if (start_pos < 0) return arg_error("attention_q8: start_pos must not be negative");
    if (!kc || !ks || !vc || !vs || cap <= 0) return arg_error("attention_q8: KV cache pointers incomplete");
    if ((long long)start_pos + seq > cap) {
        set_error("attention_q8: KV cache capacity exceeded");
        return JYC_ERR_KV_OOM;
    }
    if (!Q || !K || !V || !out) return arg_error("attention_q8: null pointer");
    if (head_dim % 4 || head_dim > 256) return arg_error("attention_q8: head_dim must be a multiple of 4, <= 256");
    cudaStream_t s = S(stream);
    const int rows_max = 8;
    if (attn_smem_bytes(rows_max, num_heads, num_kv_heads, head_dim) > 200 * 1024)
        return arg_error("attention_q8: query-head group too large");
    KVView kv{kc, ks, vc, vs, (long long)num_kv_heads * head_dim, head_dim, num_kv_heads, 1, cap};
    const int maxpos = start_pos + seq;
    const int target = std::max(1, 296 / num_kv_heads);
    int chunk = (maxpos + target - 1) / target;
    chunk = std::max(64, (chunk + 63) / 64 * 64);
    const int nsplit = (maxpos + chunk - 1) / chunk;
    Scratch sc(s);
    int8_t* q8;
    float *qsc, *po, *pml;
    unsigned int* arrive;
    TRY(sc.get(&q8, (size_t)rows_max * num_heads * head_dim));
    TRY(sc.get(&qsc, (size_t)rows_max * num_heads));
    TRY(sc.get(&po, (size_t)rows_max * num_heads * nsplit * head_dim));
    TRY(sc.get(&pml, (size_t)rows_max * num_heads * nsplit * 2));
    TRY(sc.get(&arrive, (size_t)num_kv_heads));
    JYC_CUDA(cudaMemsetAsync(arrive, 0, num_kv_heads * sizeof(unsigned int), s));
    const int qd = num_heads * head_dim, kvd = num_kv_heads * head_dim;
    for (int r0 = 0; r0 < seq; r0 += rows_max) {
        const int rows = std::min(rows_max, seq - r0);
        // kv_pack_q8 of the new K,V rows into the cache + Q quantisation (inputs already roped)
        RopeQuantArgs rq{};
        rq.q = Q + (size_t)r0 * qd; rq.k = K + (size_t)r0 * kvd; rq.v = V + (size_t)r0 * kvd;
        rq.ldq = 0;  // set per array below
        rq.rows = rows; rq.H = num_heads; rq.KV = num_kv_heads; rq.hd = head_dim;
        rq.q8 = q8; rq.qsc = qsc; rq.kv = kv; rq.pos = PosSrc{nullptr, start_pos + r0};
        // Q, K, V have different row strides: run Q-only and K/V-only passes.
        {
            RopeQuantArgs a = rq;  // queries: H heads, stride qd
            a.KV = 0; a.ldq = qd;
            // with KV = 0 the kernel only visits query heads
            TRY(launch_rope_quant(a, s));
        }
        {
            RopeQuantArgs a = rq;  // keys and values: stride kvd, no query heads
            a.H = 0; a.ldq = kvd;
            a.q8 = nullptr; a.qsc = nullptr;
            TRY(launch_rope_quant(a, s));
        }
        AttnArgs at{};
        at.q8 = q8; at.qsc = qsc; at.kv = kv;
        at.rows = rows; at.H = num_heads; at.KV = num_kv_heads; at.hd = head_dim;
        at.chunk = chunk; at.nsplit = nsplit; at.scale = 1.0f / sqrtf((float)head_dim);
        at.part_o = po; at.part_ml = pml; at.arrive = arrive;
        at.out = out + (size_t)r0 * qd; at.ldo = qd; at.pos = PosSrc{nullptr, start_pos + r0};
        TRY(launch_attention(at, s));
    }
    return JYC_OK;
}

// ---------------------------------------------------------------------------
// jyc_attention_q8_noalloc: the same kernels with a fixed scratch array.
}  // extern "C"

namespace {

constexpr size_t kNaQ8 = 8 * 8192;        // int8 queries: 8 rows x num_heads*head_dim
constexpr size_t kNaQsc = 8 * 1024;       // floats: 8 rows x num_heads
constexpr size_t kNaPo = 1u << 20;        // floats: split partial outputs (4 MiB)
constexpr size_t kNaPml = 1u << 16;       // floats: split (max, sum) pairs
constexpr size_t kNaArrive = 256;         // uint32 arrival counters, one per kv head
constexpr size_t kNaBytes = kNaQ8 + (kNaQsc + kNaPo + kNaPml) * 4 + kNaArrive * 4;
static __device__ __align__(256) unsigned char g_noalloc_scratch[kNaBytes];

// address of the array on each device, resolved once with that device current
std::mutex g_na_mu;
std::vector<unsigned char*> g_na_addr;

int noalloc_scratch(unsigned char** out) {
    int dev = 0;
    JYC_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lk(g_na_mu);
    if ((int)g_na_addr.size() <= dev) g_na_addr.resize(dev + 1, nullptr);
    if (!g_na_addr[dev]) {
        void* p = nullptr;
        JYC_CUDA(cudaGetSymbolAddress(&p, g_noalloc_scratch));
        g_na_addr[dev] = static_cast<unsigned char*>(p);
    }
    *out = g_na_addr[dev];
    return JYC_OK;
}

}  // namespace

extern "C" {

JYC_API int jyc_attention_q8_noalloc(const float* Q, const float* K, const float* V, float* out, int seq,
                                     int start_pos, int num_heads, int num_kv_heads, int head_dim,
                                     int8_t* kc, float* ks, int8_t* vc, float* vs, int cap, void* stream) {
    clear_error();
    if (num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
        return arg_error("attention_q8_noalloc: num_heads must be a multiple of num_kv_heads");
    if (seq <= 0) return arg_error("attention_q8_noalloc: seq must be positive");
    if (start_pos < 0) return arg_error("attention_q8_noalloc: start_pos must not be negative");
    if (!kc || !ks || !vc || !vs || cap <= 0) return arg_error("attention_q8_noalloc: KV cache pointers incomplete");
    if ((long long)start_pos + seq > cap) {
        set_error("attention_q8_noalloc: KV cache capacity exceeded");
        return JYC_ERR_KV_OOM;
    }
    if (!Q || !K || !V || !out) return arg_error("attention_q8_noalloc: null pointer");
    if (head_dim % 4 || head_dim > 256)
        return arg_error("attention_q8_noalloc: head_dim must be a multiple of 4, <= 256");
    const int rows_max = 8;
    if (attn_smem_bytes(rows_max, num_heads, num_kv_heads, head_dim) > 200 * 1024)
        return arg_error("attention_q8_noalloc: query-head group too large");
    const int maxpos = start_pos + seq;
    const int target = std::max(1, 296 / num_kv_heads);
    int chunk = (maxpos + target - 1) / target;
    chunk = std::max(64, (chunk + 63) / 64 * 64);
    const int nsplit = (maxpos + chunk - 1) / chunk;
    const size_t need_q8 = (size_t)rows_max * num_heads * head_dim;
    const size_t need_qsc = (size_t)rows_max * num_heads;
    const size_t need_po = (size_t)rows_max * num_heads * nsplit * head_dim;
    const size_t need_pml = (size_t)rows_max * num_heads * nsplit * 2;
    if (need_q8 > kNaQ8 || need_qsc > kNaQsc || need_po > kNaPo || need_pml > kNaPml ||
        (size_t)num_kv_heads > kNaArrive)
        return arg_error("attention_q8_noalloc: call exceeds the fixed scratch (num_heads*head_dim <= 8192, "
                         "num_kv_heads <= 256, 8*num_heads*head_dim*splits <= 1048576 floats)");
    unsigned char* base = nullptr;
    TRY(noalloc_scratch(&base));
    int8_t* q8 = reinterpret_cast<int8_t*>(base);
    float* qsc = reinterpret_cast<float*>(base + kNaQ8);
    float* po = qsc + kNaQsc;
    float* pml = po + kNaPo;
    unsigned int* arrive = reinterpret_cast<unsigned int*>(pml + kNaPml);
    cudaStream_t s = S(stream);
    KVView kv{kc, ks, vc, vs, (long long)num_kv_heads * head_dim, head_dim, num_kv_heads, 1, cap};
    const int qd = num_heads * head_dim, kvd = num_kv_heads * head_dim;
    for (int r0 = 0; r0 < seq; r0 += rows_max) {
        const int rows = std::min(rows_max, seq - r0);
        RopeQuantArgs rq{};
        rq.q = Q + (size_t)r0 * qd; rq.k = K + (size_t)r0 * kvd; rq.v = V + (size_t)r0 * kvd;
        rq.rows = rows; rq.H = num_heads; rq.KV = num_kv_heads; rq.hd = head_dim;
        rq.q8 = q8; rq.qsc = qsc; rq.kv = kv; rq.pos = PosSrc{nullptr, start_pos + r0};
        {
            RopeQuantArgs a = rq;
            a.KV = 0; a.ldq = qd;
            TRY(launch_rope_quant(a, s));
        }
        {
            RopeQuantArgs a = rq;
            a.H = 0; a.ldq = kvd;
            a.q8 = nullptr; a.qsc = nullptr;
            TRY(launch_rope_quant(a, s));
        }
        AttnArgs at{};
        at.q8 = q8; at.qsc = qsc; at.kv = kv;
        at.rows = rows; at.H = num_heads; at.KV = num_kv_heads; at.hd = head_dim;
        at.chunk = chunk; at.nsplit = nsplit; at.scale = 1.0f / sqrtf((float)head_dim);
        at.part_o = po; at.part_ml = pml; at.arrive = arrive;
        at.out = out + (size_t)r0 * qd; at.ldo = qd; at.pos = PosSrc{nullptr, start_pos + r0};
        TRY(launch_attention(at, s));
    }
    return JYC_OK;
}

JYC_API int jyc_silu(const float* x, float* y, int n, void* stream) {
    clear_error();
    if ((!x || !y) && n > 0) return arg_error("silu: null pointer");
    return launch_silu(x, y, n, S(stream));
}

JYC_API int jyc_argmax(const float* logits, int n, int* out_index, void* stream) {
    clear_error();
    if (!logits || !out_index) return arg_error("argmax: null pointer");
    cudaStream_t s = S(stream);
    Scratch sc(s);
    unsigned long long* slot;
    TRY(sc.get(&slot, 1));
    JYC_CUDA(cudaMemsetAsync(slot, 0, sizeof(unsigned long long), s));
    return launch_argmax(logits, n, slot, out_index, s);
}

JYC_API int jyc_sample(float* logits, int vocab_size, float temperature, float repetition_penalty,
                       const int* out_ids, int prompt_len, int len, unsigned int* rng, int* next, void* stream) {
    clear_error();
    if (!logits || !rng || !next || vocab_size <= 0) return arg_error("sample: bad arguments");
    if (repetition_penalty != 1.0f && (!out_ids || prompt_len < 0 || len < prompt_len))
        return arg_error("sample: penalty needs out_ids[prompt_len..len)");
    return launch_sample(logits, vocab_size, temperature, repetition_penalty, out_ids, prompt_len, len, rng, next,
                         S(stream));
}

// ---------------------------------------------------------------------------
// Paged K/V cache and batched sampling.
}  // extern "C"

namespace {

// The arguments that the paged operators share; `what` names the caller.
int check_paged(const char* what, int num_kv_heads, int head_dim, const int* page_table, int table_stride,
                int num_seqs, const jyc_kv_pages* p) {
    auto bad = [&](const char* msg) { return arg_error(std::string(what) + ": " + msg); };
    if (num_kv_heads <= 0) return bad("num_kv_heads must be positive");
    if (head_dim <= 0 || head_dim % 4 || head_dim > 256) return bad("head_dim must be a multiple of 4, <= 256");
    if (num_seqs < 0 || table_stride < 0) return bad("negative page table shape");
    if (!page_table || !p || !p->k || !p->ks || !p->v || !p->vs) return bad("null pointer");
    if (p->num_pages <= 0 || p->page_size <= 0) return bad("num_pages and page_size must be positive");
    if ((long long)table_stride * p->page_size > 0x7fffff00LL)
        return bad("table_stride * page_size must be below 2^31 - 255");
    if (p->page_stride < 0 || p->pos_stride < 0 || p->head_stride < 0 || p->spage_stride < 0 || p->spos_stride < 0 ||
        p->shead_stride < 0)
        return bad("negative page stride");
    if ((((uintptr_t)p->k | (uintptr_t)p->v) & 3) || ((p->page_stride | p->pos_stride | p->head_stride) & 3))
        return bad("k, v and their strides must be multiples of 4 bytes");
    if (((uintptr_t)p->ks | (uintptr_t)p->vs | (uintptr_t)page_table) & 3) return bad("misaligned scales or page table");
    return JYC_OK;
}

int check_rope(const char* what, const float* cos_table, const float* sin_table, int rope_len) {
    if (!cos_table != !sin_table) return arg_error(std::string(what) + ": cos and sin tables come together");
    if (cos_table && rope_len <= 0) return arg_error(std::string(what) + ": rope_len must be positive");
    return JYC_OK;
}

}  // namespace

extern "C" {

JYC_API int jyc_kv_append_paged_q8(const float* K, const float* V, int ld, int rows, int num_kv_heads, int head_dim,
                                   const int* row_seq, const int* row_pos, const int* page_table, int table_stride,
                                   int num_seqs, const float* cos_table, const float* sin_table, int rope_len,
                                   const jyc_kv_pages* pages, void* stream) {
    clear_error();
    TRY(check_paged("kv_append_paged_q8", num_kv_heads, head_dim, page_table, table_stride, num_seqs, pages));
    TRY(check_rope("kv_append_paged_q8", cos_table, sin_table, rope_len));
    if (rows < 0) return arg_error("kv_append_paged_q8: negative rows");
    if (ld < (long long)num_kv_heads * head_dim) return arg_error("kv_append_paged_q8: ld below num_kv_heads * head_dim");
    if (!row_seq && rows > num_seqs) return arg_error("kv_append_paged_q8: more rows than sequences without row_seq");
    if (rows == 0) return JYC_OK;
    if (!K || !V || !row_pos) return arg_error("kv_append_paged_q8: null pointer");
    const PagedKV kv{*pages, page_table, table_stride, num_seqs, fast_div(pages->page_size)};
    return launch_paged_append(K, V, ld, rows, num_kv_heads, head_dim, row_seq, row_pos, kv,
                               PagedRope{cos_table, sin_table, rope_len}, S(stream));
}

JYC_API int jyc_kv_read_paged_q8(float* K, float* V, int ld, int rows, int num_kv_heads, int head_dim,
                                 const int* row_seq, const int* row_pos, const int* page_table, int table_stride,
                                 int num_seqs, const jyc_kv_pages* pages, void* stream) {
    clear_error();
    TRY(check_paged("kv_read_paged_q8", num_kv_heads, head_dim, page_table, table_stride, num_seqs, pages));
    if (rows < 0) return arg_error("kv_read_paged_q8: negative rows");
    if (ld < (long long)num_kv_heads * head_dim) return arg_error("kv_read_paged_q8: ld below num_kv_heads * head_dim");
    if (!row_seq && rows > num_seqs) return arg_error("kv_read_paged_q8: more rows than sequences without row_seq");
    if (rows == 0) return JYC_OK;
    if (!K || !V || !row_pos) return arg_error("kv_read_paged_q8: null pointer");
    const PagedKV kv{*pages, page_table, table_stride, num_seqs, fast_div(pages->page_size)};
    return launch_paged_read(K, V, ld, rows, num_kv_heads, head_dim, row_seq, row_pos, kv, S(stream));
}

JYC_API size_t jyc_attention_paged_q8_workspace(int num_seqs, int num_heads, int num_kv_heads, int head_dim) {
    clear_error();
    if (num_seqs < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || head_dim <= 0 ||
        head_dim % 4 || head_dim > 256) {
        arg_error("attention_paged_q8_workspace: bad shape");
        return 0;
    }
    return paged_attention_workspace(num_heads, num_kv_heads, head_dim);
}

JYC_API int jyc_attention_paged_q8(const float* Q, int ldq, float* out, int ldo, int num_heads, int num_kv_heads,
                                   int head_dim, const int* seq_lens, const int* page_table, int table_stride,
                                   int num_seqs, const float* cos_table, const float* sin_table, int rope_len,
                                   const jyc_kv_pages* pages, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    TRY(check_paged("attention_paged_q8", num_kv_heads, head_dim, page_table, table_stride, num_seqs, pages));
    TRY(check_rope("attention_paged_q8", cos_table, sin_table, rope_len));
    if (num_heads <= 0 || num_heads % num_kv_heads)
        return arg_error("attention_paged_q8: num_heads must be a multiple of num_kv_heads");
    if (ldq < (long long)num_heads * head_dim || ldo < (long long)num_heads * head_dim)
        return arg_error("attention_paged_q8: ldq and ldo must hold num_heads * head_dim");
    if (num_seqs == 0) return JYC_OK;
    if (!Q || !out || !seq_lens) return arg_error("attention_paged_q8: null pointer");
    const size_t need = paged_attention_workspace(num_heads, num_kv_heads, head_dim);
    if (need == 0) return JYC_ERR_CUDA;
    if (workspace && workspace_bytes < need) return arg_error("attention_paged_q8: workspace too small");
    if ((uintptr_t)workspace & 15) return arg_error("attention_paged_q8: workspace must be 16-byte aligned");
    PagedAttn a{};
    a.Q = Q; a.ldq = ldq; a.out = out; a.ldo = ldo;
    a.H = num_heads; a.KV = num_kv_heads; a.hd = head_dim; a.lens = seq_lens;
    a.kv = PagedKV{*pages, page_table, table_stride, num_seqs, fast_div(pages->page_size)};
    a.rope = PagedRope{cos_table, sin_table, rope_len};
    a.scale = 1.0f / sqrtf((float)head_dim);
    Scratch sc(S(stream));
    unsigned char* own = nullptr;
    if (!workspace) TRY(sc.get(&own, need));
    return launch_paged_attention(a, workspace ? workspace : own, S(stream));
}

JYC_API int jyc_paged_error(int reset) {
    clear_error();
    int* p = paged_error_word();
    if (!p) {
        set_error("paged_error: no device");
        return JYC_ERR_CUDA;
    }
    int v = 0;
    JYC_CUDA(cudaDeviceSynchronize());
    JYC_CUDA(cudaMemcpy(&v, p, sizeof(int), cudaMemcpyDeviceToHost));
    if (reset && v) TRY(paged_error_clear(v));
    return v;
}

JYC_API int jyc_sample_batch(const float* logits, int ld, int rows, int vocab_size, const float* temperature,
                             const int* top_k, const float* top_p, const float* min_p, const float* u, int* out_ids,
                             float* out_probs, void* stream) {
    clear_error();
    if (rows < 0 || vocab_size <= 0) return arg_error("sample_batch: need rows >= 0 and vocab_size > 0");
    if (vocab_size > kPickMaxVocab) return arg_error("sample_batch: vocab_size above 2^20");
    if (ld < vocab_size) return arg_error("sample_batch: ld below vocab_size");
    if (rows == 0) return JYC_OK;
    if (!logits || !u || !out_ids) return arg_error("sample_batch: null pointer");
    const PickArgs a{logits, ld, rows, vocab_size, temperature, top_k, top_p, min_p, u, out_ids, out_probs};
    return launch_pick(a, S(stream));
}

}  // extern "C"

// ---------------------------------------------------------------------------
// Rotary rows, 8-bit products and the 4-bit paged cache.
namespace {

// Whether an array of 4-byte numbers does not lie on 4 bytes.
template <class... P>
bool askew(P... p) {
    return ((0 | ... | (uintptr_t)p) & 3) != 0;
}

int check_rope_view(const char* what, const jyc_rope* r, int head_dim, RopeView* v) {
    auto bad = [&](const char* msg) { return arg_error(std::string(what) + ": " + msg); };
    *v = RopeView{nullptr, nullptr, 0, 0, false};
    if (!r) return JYC_OK;
    if (!r->cos_table || !r->sin_table) return bad("cos and sin tables come together");
    if (((uintptr_t)r->cos_table | (uintptr_t)r->sin_table) & 3) return bad("misaligned tables");
    if (r->len <= 0) return bad("the tables' len must be positive");
    if (r->rot_dim <= 0 || r->rot_dim % 2 || r->rot_dim > head_dim) return bad("rot_dim must be even, <= head_dim");
    if (r->layout != JYC_ROPE_PAIRS && r->layout != JYC_ROPE_HALVES) return bad("unknown rope layout");
    *v = RopeView{r->cos_table, r->sin_table, r->len, r->rot_dim / 2, r->layout == JYC_ROPE_HALVES};
    return JYC_OK;
}

// The arguments that the operators of the 4-bit pages share.
int check_paged4(const char* what, int num_kv_heads, int head_dim, const int* page_table, int table_stride,
                 int num_seqs, const jyc_kv_pages_q4* p) {
    auto bad = [&](const char* msg) { return arg_error(std::string(what) + ": " + msg); };
    if (num_kv_heads <= 0) return bad("num_kv_heads must be positive");
    if (head_dim <= 0 || head_dim % 4 || head_dim > 256) return bad("head_dim must be a multiple of 4, <= 256");
    if (num_seqs < 0 || table_stride < 0) return bad("negative page table shape");
    if (!page_table || !p || !p->k || !p->kp || !p->v || !p->vp) return bad("null pointer");
    if (p->num_pages <= 0 || p->page_size <= 0) return bad("num_pages and page_size must be positive");
    if ((long long)table_stride * p->page_size > 0x7fffff00LL)
        return bad("table_stride * page_size must be below 2^31 - 255");
    if (p->page_stride < 0 || p->pos_stride < 0 || p->head_stride < 0 || p->ppage_stride < 0 || p->ppos_stride < 0 ||
        p->phead_stride < 0 || p->mpage_stride < 0 || p->mpos_stride < 0 || p->mhead_stride < 0)
        return bad("negative page stride");
    if ((((uintptr_t)p->k | (uintptr_t)p->v) & 15) || ((p->page_stride | p->pos_stride | p->head_stride) & 15))
        return bad("k, v and their strides must be multiples of 16 bytes");
    if (((uintptr_t)p->kp | (uintptr_t)p->vp | (uintptr_t)p->mass | (uintptr_t)page_table) & 3)
        return bad("misaligned parameters, mass or page table");
    return JYC_OK;
}

// Of one launch's grid: heads of sequences.
constexpr long long kMaxItems = 0x7fffffffLL;

// Whether a size_t counts the scores that attention leaves for its weights: a float per place of a sequence and query
// head, of which a kv head's are rounded up to 16 at most.
bool scores_countable(int num_seqs, int num_heads, int capacity) {
    return (double)num_seqs * num_heads * (capacity + 64.0) * (16 * sizeof(float)) < 9e18;
}

int paged4_view(const jyc_kv_pages_q4* pages, const int* page_table, int table_stride, int num_seqs, PagedKV4* kv) {
    int* err = paged_error_word();
    if (!err) return cuda_fail(cudaErrorNoDevice, "paged error word");
    *kv = PagedKV4{*pages, page_table, table_stride, num_seqs, fast_div(pages->page_size), err};
    return JYC_OK;
}

}  // namespace

extern "C" {

JYC_API int jyc_rope_rows(const float* X, int ldx, float* Y, int ldy, int rows, int num_heads, int head_dim,
                          const int* row_pos, const jyc_rope* rope, void* stream) {
    clear_error();
    if (rows < 0 || num_heads <= 0 || head_dim <= 0) return arg_error("rope_rows: bad shape");
    if (!rope) return arg_error("rope_rows: null rope");
    RopeView r;
    TRY(check_rope_view("rope_rows", rope, head_dim, &r));
    if ((long long)num_heads * head_dim > ldx || (long long)num_heads * head_dim > ldy)
        return arg_error("rope_rows: ldx and ldy must hold num_heads * head_dim");
    if (rows == 0) return JYC_OK;
    if (!X || !Y || !row_pos) return arg_error("rope_rows: null pointer");
    if (askew(X, Y, row_pos)) return arg_error("rope_rows: misaligned array");
    if (X == Y && ldx != ldy) return arg_error("rope_rows: in place needs ldx == ldy");
    return launch_rope_rows(X, ldx, Y, ldy, rows, num_heads, head_dim, row_pos, r, S(stream));
}

JYC_API int jyc_quantize_rows_i8(const float* x, int ldx, int rows, int k, int8_t* q, int ldq, float* scale,
                                 void* stream) {
    clear_error();
    if (rows < 0 || k <= 0) return arg_error("quantize_rows_i8: need rows >= 0 and k > 0");
    if (k > 0x7ffffc00) return arg_error("quantize_rows_i8: k must be at most 2^31 - 1024");
    if (ldx < k || ldq < k) return arg_error("quantize_rows_i8: ldx and ldq must hold k");
    if (rows == 0) return JYC_OK;
    if (!x || !q || !scale) return arg_error("quantize_rows_i8: null pointer");
    if (askew(x, scale)) return arg_error("quantize_rows_i8: misaligned array");
    return launch_quantize_rows(x, ldx, rows, k, q, ldq, scale, S(stream));
}

JYC_API int jyc_matmul_i8(const int8_t* A, int lda, const float* a_scale, const int8_t* W, int ldw,
                          const float* w_scale, const float* bias, float* C, int ldc, int m, int n, int k,
                          void* stream) {
    clear_error();
    if (m < 0 || n <= 0 || k <= 0) return arg_error("matmul_i8: need m >= 0 and n, k > 0");
    if (k > 131071) return arg_error("matmul_i8: k above 131071 can pass 32-bit sums");
    if (m > 0x7fffff00 || n > 0x7fffff00) return arg_error("matmul_i8: m and n must be at most 2^31 - 256");
    if (lda < k || ldw < k || ldc < n) return arg_error("matmul_i8: lda and ldw must hold k, ldc must hold n");
    if ((lda | ldw) & 15) return arg_error("matmul_i8: lda and ldw must be multiples of 16");
    if (m == 0) return JYC_OK;
    if (!A || !a_scale || !W || !w_scale || !C) return arg_error("matmul_i8: null pointer");
    if (askew(a_scale, w_scale, bias, C)) return arg_error("matmul_i8: misaligned array");
    if (((uintptr_t)A | (uintptr_t)W) & 15) return arg_error("matmul_i8: A and W must be 16-byte aligned");
    return launch_i8_gemm(I8Gemm{A, lda, a_scale, W, ldw, w_scale, bias, C, ldc, m, n, k}, S(stream));
}

JYC_API int jyc_kv_append_paged_q4(const float* K, const float* V, int ld, int rows, int num_kv_heads, int head_dim,
                                   const int* row_seq, const int* row_pos, const int* page_table, int table_stride,
                                   int num_seqs, const jyc_rope* rope, const int* rope_pos,
                                   const jyc_kv_pages_q4* pages, void* stream) {
    clear_error();
    TRY(check_paged4("kv_append_paged_q4", num_kv_heads, head_dim, page_table, table_stride, num_seqs, pages));
    RopeView r;
    TRY(check_rope_view("kv_append_paged_q4", rope, head_dim, &r));
    if (rows < 0) return arg_error("kv_append_paged_q4: negative rows");
    if (ld < (long long)num_kv_heads * head_dim) return arg_error("kv_append_paged_q4: ld below num_kv_heads * head_dim");
    if (!row_seq && rows > num_seqs) return arg_error("kv_append_paged_q4: more rows than sequences without row_seq");
    if (rows == 0) return JYC_OK;
    if (!K || !V || !row_pos) return arg_error("kv_append_paged_q4: null pointer");
    if (askew(K, V, row_seq, row_pos, rope_pos)) return arg_error("kv_append_paged_q4: misaligned array");
    PagedKV4 kv;
    TRY(paged4_view(pages, page_table, table_stride, num_seqs, &kv));
    return launch_paged4_append(K, V, ld, rows, num_kv_heads, head_dim, row_seq, row_pos, rope_pos, kv, r, S(stream));
}

JYC_API int jyc_kv_read_paged_q4(float* K, float* V, int ld, int rows, int num_kv_heads, int head_dim,
                                 const int* row_seq, const int* row_pos, const int* page_table, int table_stride,
                                 int num_seqs, const jyc_kv_pages_q4* pages, void* stream) {
    clear_error();
    TRY(check_paged4("kv_read_paged_q4", num_kv_heads, head_dim, page_table, table_stride, num_seqs, pages));
    if (rows < 0) return arg_error("kv_read_paged_q4: negative rows");
    if (ld < (long long)num_kv_heads * head_dim) return arg_error("kv_read_paged_q4: ld below num_kv_heads * head_dim");
    if (!row_seq && rows > num_seqs) return arg_error("kv_read_paged_q4: more rows than sequences without row_seq");
    if (rows == 0) return JYC_OK;
    if (!K || !V || !row_pos) return arg_error("kv_read_paged_q4: null pointer");
    if (askew(K, V, row_seq, row_pos)) return arg_error("kv_read_paged_q4: misaligned array");
    PagedKV4 kv;
    TRY(paged4_view(pages, page_table, table_stride, num_seqs, &kv));
    return launch_paged4_read(K, V, ld, rows, num_kv_heads, head_dim, row_seq, row_pos, kv, S(stream));
}

JYC_API size_t jyc_attention_paged_q4_workspace(int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                                                int capacity) {
    clear_error();
    if (num_seqs < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || head_dim <= 0 ||
        head_dim % 4 || head_dim > 256 || capacity < 0 || capacity > 0x7fffff00 ||
        (long long)num_seqs * num_heads > kMaxItems || !scores_countable(num_seqs, num_heads, capacity)) {
        arg_error("attention_paged_q4_workspace: bad shape");
        return 0;
    }
    const size_t n = paged4_attention_workspace(num_seqs, num_heads, num_kv_heads, head_dim, capacity);
    if (n == 0) cuda_fail(cudaErrorNoDevice, "attention_paged_q4_workspace: device query");
    return n;
}

JYC_API int jyc_attention_paged_q4(const float* Q, int ldq, float* out, int ldo, int num_heads, int num_kv_heads,
                                   int head_dim, const int* seq_lens, const int* page_table, int table_stride,
                                   int num_seqs, const jyc_rope* rope, const int* rope_pos,
                                   const jyc_kv_pages_q4* pages, void* workspace, size_t workspace_bytes,
                                   void* stream) {
    clear_error();
    TRY(check_paged4("attention_paged_q4", num_kv_heads, head_dim, page_table, table_stride, num_seqs, pages));
    RopeView r;
    TRY(check_rope_view("attention_paged_q4", rope, head_dim, &r));
    if (num_heads <= 0 || num_heads % num_kv_heads)
        return arg_error("attention_paged_q4: num_heads must be a multiple of num_kv_heads");
    if (ldq < (long long)num_heads * head_dim || ldo < (long long)num_heads * head_dim)
        return arg_error("attention_paged_q4: ldq and ldo must hold num_heads * head_dim");
    if ((long long)num_seqs * num_heads > kMaxItems) return arg_error("attention_paged_q4: num_seqs * num_heads above 2^31 - 1");
    if (num_seqs == 0) return JYC_OK;
    if (!Q || !out || !seq_lens) return arg_error("attention_paged_q4: null pointer");
    if (askew(Q, out, seq_lens, rope_pos)) return arg_error("attention_paged_q4: misaligned array");
    const int capacity = pages->mass ? table_stride * pages->page_size : 0;
    if (!scores_countable(num_seqs, num_heads, capacity)) return arg_error("attention_paged_q4: too many places for a workspace");
    const size_t need = paged4_attention_workspace(num_seqs, num_heads, num_kv_heads, head_dim, capacity);
    if (need == 0) return cuda_fail(cudaErrorNoDevice, "attention_paged_q4: device query");
    if (workspace && workspace_bytes < need) return arg_error("attention_paged_q4: workspace too small");
    if ((uintptr_t)workspace & 15) return arg_error("attention_paged_q4: workspace must be 16-byte aligned");
    PagedAttn4 a{};
    a.Q = Q; a.ldq = ldq; a.out = out; a.ldo = ldo;
    a.H = num_heads; a.KV = num_kv_heads; a.hd = head_dim; a.lens = seq_lens; a.rope_pos = r.cos_t ? rope_pos : nullptr;
    TRY(paged4_view(pages, page_table, table_stride, num_seqs, &a.kv));
    a.rope = r;
    a.scale = 1.0f / sqrtf((float)head_dim);
    Scratch sc(S(stream));
    unsigned char* own = nullptr;
    if (!workspace) TRY(sc.get(&own, need));
    return launch_paged4_attention(a, workspace ? workspace : own, S(stream));
}

JYC_API int jyc_kv_evict_paged_q4(const int* seq_lens, int budget, int recent, int num_kv_heads, int head_dim,
                                  const int* page_table, int table_stride, int num_seqs, const int* new_table,
                                  int new_stride, int* new_lens, int* kept, const jyc_kv_pages_q4* pages,
                                  void* stream) {
    clear_error();
    TRY(check_paged4("kv_evict_paged_q4", num_kv_heads, head_dim, page_table, table_stride, num_seqs, pages));
    if (budget <= 0 || recent < 0 || recent > budget) return arg_error("kv_evict_paged_q4: need 0 <= recent <= budget, budget > 0");
    if (!pages->mass) return arg_error("kv_evict_paged_q4: the pages have no mass");
    if (new_stride < 0 || (long long)new_stride * pages->page_size < budget || (long long)new_stride * pages->page_size > 0x7fffff00LL)
        return arg_error("kv_evict_paged_q4: new_stride * page_size must hold the budget, below 2^31 - 255");
    if ((long long)num_seqs * num_kv_heads > (1LL << 30) / budget)
        return arg_error("kv_evict_paged_q4: num_seqs * num_kv_heads * budget above 2^30");
    if (num_seqs == 0) return JYC_OK;
    if (!seq_lens || !new_table || !new_lens || !kept) return arg_error("kv_evict_paged_q4: null pointer");
    if (askew(seq_lens, new_table, new_lens, kept)) return arg_error("kv_evict_paged_q4: misaligned array");
    if (seq_lens == new_lens) return arg_error("kv_evict_paged_q4: new_lens must be another array than seq_lens");
    PagedEvict4 e{};
    e.lens = seq_lens; e.budget = budget; e.recent = recent; e.KV = num_kv_heads; e.hd = head_dim;
    TRY(paged4_view(pages, page_table, table_stride, num_seqs, &e.kv));
    e.new_table = new_table; e.new_stride = new_stride; e.new_lens = new_lens; e.kept = kept;
    return launch_paged4_evict(e, S(stream));
}

}  // extern "C"
