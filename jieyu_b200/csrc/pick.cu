// pick.cu — the next token of every row of a batch: temperature, top-k, top-p
// and min-p filters, then one inverse-CDF draw per row from a given random
// number (beside sample.cuh, which restates the reference's one-row sampler).
//
// Weights w = exp((l - max) / T) are held as 2^42 fixed point in 64 bits
// (below 2^-40: zero), so every sum of them is the same in any order.
#include "paged.cuh"

namespace jyc {

namespace {

constexpr int kPickThreads = 1024;

__device__ __forceinline__ uint32_t pick_key(float l) { return f32_order_key(l + 0.0f); }  // -0 -> +0

__device__ __forceinline__ double pick_w(float l, float mx, double T) {
    if (l == mx) return 1.0;
    if (!(l > -INFINITY)) return 0.0;
    const double w = exp(((double)l - (double)mx) / T);
    return w < 0x1p-40 ? 0.0 : w;
}
__device__ __forceinline__ unsigned long long pick_fix(double w) { return (unsigned long long)rint(w * 0x1p42); }

// exclusive sum over the block of one value per thread; *total: all of them
template <class T>
__device__ T block_scan(T v, T* s, T* total) {
    const int tid = threadIdx.x;
    s[tid] = v;
    __syncthreads();
    for (int o = 1; o < kPickThreads; o <<= 1) {
        const T x = tid >= o ? s[tid - o] : T(0);
        __syncthreads();
        s[tid] += x;
        __syncthreads();
    }
    *total = s[kPickThreads - 1];
    const T r = s[tid] - v;
    __syncthreads();
    return r;
}

// One CTA per row; thread t owns a contiguous run of the vocabulary.
__global__ void __launch_bounds__(kPickThreads) pick_kernel(PickArgs a) {
    __shared__ unsigned long long s_scan[kPickThreads];
    __shared__ unsigned long long s_mass[256];
    __shared__ unsigned int s_cnt[256];
    __shared__ unsigned int s_key;
    __shared__ unsigned long long s_rest;
    const int row = blockIdx.x, tid = threadIdx.x, V = a.V;
    const float* l = a.logits + (size_t)row * a.ld;
    const int per = (V + kPickThreads - 1) / kPickThreads, v0 = min(V, tid * per), v1 = min(V, v0 + per);

    // first index of the maximum
    unsigned long long best = 0ull;
    for (int v = v0; v < v1; v++) best = max(best, argmax_pack(l[v] + 0.0f, v));
    s_scan[tid] = best;
    __syncthreads();
    for (int o = kPickThreads / 2; o > 0; o >>= 1) {
        if (tid < o) s_scan[tid] = max(s_scan[tid], s_scan[tid + o]);
        __syncthreads();
    }
    best = s_scan[0];
    __syncthreads();
    const int first = argmax_index(best);
    const float mx = (best >> 32) ? l[first] + 0.0f : -INFINITY;
    const float Tf = a.temperature ? a.temperature[row] : 1.0f;
    if (!(mx > -INFINITY) || !(Tf > 0.0f)) {
        if (tid == 0) {
            const bool dead = !(mx > -INFINITY);
            a.ids[row] = dead ? -1 : first;
            if (a.probs) a.probs[row] = dead ? 0.0f : 1.0f;
        }
        return;
    }
    const double T = (double)Tf;
    const int K = a.top_k ? a.top_k[row] : 0;
    const float P = a.top_p ? a.top_p[row] : 1.0f;
    const double mp = a.min_p ? fmin((double)a.min_p[row], 1.0) : 0.0;

    // kept: keys above tau, and the first `ties` (by index) equal to it
    uint32_t tau = 0u;
    unsigned long long ties = ~0ull;
    if (K > 0 && K < V) {
        uint32_t prefix = 0u;
        unsigned long long rest = (unsigned long long)K;
        for (int sh = 24; sh >= 0; sh -= 8) {
            if (tid < 256) s_cnt[tid] = 0u;
            __syncthreads();
            const uint32_t hi = sh == 24 ? 0u : ~0u << (sh + 8);
            for (int v = v0; v < v1; v++) {
                const uint32_t k = pick_key(l[v]);
                if ((k & hi) == prefix) atomicAdd(&s_cnt[(k >> sh) & 255], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                int d = 255;
                while (s_cnt[d] < rest) rest -= s_cnt[d--];
                s_key = prefix | ((uint32_t)d << sh);
                s_rest = rest;
            }
            __syncthreads();
            prefix = s_key;
            rest = s_rest;
        }
        tau = prefix;
        ties = rest;
    }
    if (P < 1.0f) {
        // mass of the kept set, then the shortest prefix (key descending, index ascending) reaching P of it
        unsigned long long mass = 0ull, M, c;
        for (int v = v0; v < v1; v++)
            if (pick_key(l[v]) > tau) mass += pick_fix(pick_w(l[v], mx, T));
        block_scan(mass, s_scan, &M);
        if (tau != 0u) {
            unsigned long long n = 0ull;
            float lt = 0.0f;
            for (int v = v0; v < v1; v++)
                if (pick_key(l[v]) == tau) {
                    n++;
                    lt = l[v];
                }
            block_scan(n, s_scan, &c);
            block_scan(n ? pick_fix(pick_w(lt, mx, T)) * n : 0ull, s_scan, &mass);
            M += mass / c * ties;
        }
        const double need = (double)P * (double)M;
        uint32_t prefix = 0u;
        unsigned long long above = 0ull;
        for (int sh = 24; sh >= 0; sh -= 8) {
            if (tid < 256) s_mass[tid] = 0ull;
            if (tid < 256) s_cnt[tid] = 0u;
            __syncthreads();
            const uint32_t hi = sh == 24 ? 0u : ~0u << (sh + 8);
            for (int v = v0; v < v1; v++) {
                const uint32_t k = pick_key(l[v]);
                if ((k & hi) == prefix && k >= tau) {
                    atomicAdd(&s_mass[(k >> sh) & 255], pick_fix(pick_w(l[v], mx, T)));
                    atomicAdd(&s_cnt[(k >> sh) & 255], 1u);
                }
            }
            __syncthreads();
            if (tid == 0) {
                int d = 255, last = 255;
                for (; d >= 0; d--) {
                    if (s_cnt[d] == 0u) continue;
                    last = d;
                    if ((double)(above + s_mass[d]) >= need) break;
                    if (d > 0) above += s_mass[d];
                }
                d = d < 0 ? last : d;
                s_key = prefix | ((uint32_t)d << sh);
                s_rest = above;
            }
            __syncthreads();
            prefix = s_key;
            above = s_rest;
            __syncthreads();
        }
        // `above` holds the mass of keys above the border key; one of its ties at a time
        const unsigned long long n = s_cnt[prefix & 255], w = n ? s_mass[prefix & 255] / n : 0ull;
        unsigned long long m = w ? (unsigned long long)fmax(0.0, (need - (double)above) / (double)w) : 1ull;
        m = m > 1 ? m - 1 : 1;
        while (m < n && (double)(above + m * w) < need) m++;
        if (prefix > tau) {
            tau = prefix;
            ties = m;
        } else {
            ties = min(ties, m);
        }
    }
    // sums of the kept weights in index order, then the draw
    unsigned long long n = 0ull, all, sum = 0ull, total;
    if (tau != 0u)
        for (int v = v0; v < v1; v++) n += pick_key(l[v]) == tau;
    const unsigned long long before = block_scan(n, s_scan, &all);
    auto weight = [&](int v, unsigned long long& seen) {
        const uint32_t k = pick_key(l[v]);
        if (k < tau || (k == tau && tau != 0u && seen++ >= ties)) return 0ull;
        const double w = pick_w(l[v], mx, T);
        return w >= mp ? pick_fix(w) : 0ull;
    };
    unsigned long long seen = before;
    for (int v = v0; v < v1; v++) sum += weight(v, seen);
    unsigned long long cum = block_scan(sum, s_scan, &total);
    const double r = (double)a.u[row] * (double)total;
    // the first token whose running sum passes r; if none does, the last kept one
    int mine = -1;
    unsigned long long got = 0ull;
    const bool inside = sum > 0ull && !((double)cum > r) && ((double)(cum + sum) > r || cum + sum == total);
    const bool lowest = sum > 0ull && cum == 0ull && (double)cum > r;
    if (inside || lowest) {
        seen = before;
        for (int v = v0; v < v1; v++) {
            const unsigned long long w = weight(v, seen);
            if (w == 0ull) continue;
            cum += w;
            mine = v;
            got = w;
            if ((double)cum > r) break;
        }
        a.ids[row] = mine;
        if (a.probs) a.probs[row] = (float)((double)got / (double)total);
    }
}

}  // namespace

int launch_pick(const PickArgs& a, cudaStream_t s) {
    if (a.rows == 0) return JYC_OK;
    pick_kernel<<<a.rows, kPickThreads, 0, s>>>(a);
    JYC_LAUNCHED();
    return JYC_OK;
}

}  // namespace jyc
