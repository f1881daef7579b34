// paged_line.cuh — attention of one new token per sequence over a paged cache, whatever the format of its
// rows (paged.cu: 8 bits, paged4.cu: 4 bits): the line of units that all resident warps share, and the joining
// of their parts. A configuration G names the sizes (HDP, ROWS, WARPS, TK, PART, RING), the arguments (Args) and
// the usable length of a sequence (len).
#pragma once
#include "paged.cuh"
#include "ptx.cuh"

#include <cuda.h>

namespace jyc {

namespace {  // each file that includes this has its own copies

constexpr float kPaShift = 13.0f;    // the largest weight is in 2^13 .. 2^14
constexpr float kPaLow = -1.7e38f;  // reference before any key: below every score, and its differences stay finite

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// c = v + a b for a constant v, and c += a b
__device__ __forceinline__ void pa_mma_s8(const uint32_t (&a)[4], const uint32_t (&b)[2], int v, int (&c)[4]) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "r"(v));
}
__device__ __forceinline__ void pa_mma_s8(const uint32_t (&a)[4], const uint32_t (&b)[2], int (&c)[4]) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void pa_mma_f16(const uint32_t (&a)[4], const uint32_t (&b)[2], float v, float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(v));
}
__device__ __forceinline__ void pa_mma_f16(const uint32_t (&a)[4], const uint32_t (&b)[2], float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// 8 x 8 halves, lane (g, t) holding (g, 2 t) and (g, 2 t + 1), transposed
__device__ __forceinline__ uint32_t pa_transpose(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void pa_ldsm(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void pa_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// The cache is read once a step: its lines leave L2 first, so that code, queries and parts stay there
// (measured: without the hint a kernel's end runs at DRAM latency, instruction by instruction).
// Scales of neighbouring heads may share a sector, which other SMs want too: no hint.
__device__ __forceinline__ void pa_copy_scale(uint32_t dst, const float* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
template <int N>
__device__ __forceinline__ void pa_copy(uint32_t dst, const void* src, uint64_t policy) {
    if (N == 16)
        asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy)
                     : "memory");
    else
        asm volatile("cp.async.ca.shared.global.L2::cache_hint [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "l"(policy)
                     : "memory");
}
__device__ __forceinline__ uint32_t pa_pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

struct PaPlan {
    int units_row;  // kv heads * query blocks
    int qblocks;    // blocks of ROWS query heads per kv head
    int tk;         // keys of a unit
    bool wide_copy; // 16-byte copies
    bool wide_q;    // 16-byte loads of Q, 8-byte ones of the tables
    int box;        // keys of a tensor copy
    bool wide_rope; // turned4's wide form
    int team;       // warps that take the same units of neighbouring rows (where G::TEAM; units_row counts teams' rows)
};
// The line cut into runs: worker w starts at w * base + min(w, rest).
struct PaLine {
    long long base, rest, workers;
    int per_cta;  // workers of a CTA
    __device__ __forceinline__ long long start(long long w) const {
        w = min(w, workers);
        return w * base + min(w, rest);
    }
    __device__ __forceinline__ int worker(long long u) const {  // whose run holds unit u
        const long long big = rest * (base + 1);
        if (u >> 32) return (int)(u < big ? u / (base + 1) : rest + (u - big) / base);
        return (int)(u < big ? (unsigned)u / (unsigned)(base + 1) : (unsigned)rest + (unsigned)(u - big) / (unsigned)base);
    }
};
// Item that starts in a CTA and ends in a later one.
struct PaTail {
    int ctas;  // CTAs after the first that hold parts of it; 0: no such item
    int slot;  // its first part
    int b, r;
    int per_cta;
};
struct PaWork {
    PaTail* tail;      // [CTAs]
    float* part;       // [workers][2][PART]: an item's later part (0), its first (1)
    float2* stat;      // [sequence][head]: reference and 1 / sum of the weights, or nullptr
};

// Runs of U units: as many workers (warps, or teams of them) as a CTA has, or
// units; a few warps per CTA at least, whose parts are joined in shared memory.
constexpr int kPaFewWarps = 4;
__device__ __forceinline__ PaLine pa_line(long long U, int ctas, int workers, int few) {
    PaLine l;
    const long long each = U >> 31 ? workers : ((unsigned)U + ctas - 1) / (unsigned)ctas;
    l.per_cta = (int)min((long long)workers, max((long long)few, each));
    l.workers = min((long long)ctas * l.per_cta, U);
    l.base = l.rest = 0;
    if (U >> 32) {
        l.base = U / l.workers;
        l.rest = U % l.workers;
    } else if (l.workers) {
        l.base = (unsigned)U / (unsigned)l.workers;
        l.rest = (unsigned)U % (unsigned)l.workers;
    }
    return l;
}

struct PaCursor {
    int b, r, t, nt, len;  // sequence, row of units, unit and units in it, length
};
// Warps of a team, and a warp's row of units.
template <class G>
__device__ __forceinline__ int pa_team(const PaPlan& pl) {
    return G::TEAM ? pl.team : 1;
}
template <class G>
__device__ __forceinline__ int pa_row(const PaPlan& pl, const PaCursor& c) {
    const int warp = threadIdx.x >> 5;
    return G::TEAM ? c.r * pl.team + warp % pl.team : c.r;
}
template <class G>
__device__ __forceinline__ void pa_seek(const typename G::Args& a, int tk, PaCursor& c) {
    c.len = 0;
    while (c.b < a.kv.num_seqs && (c.len = G::len(a, c.b)) == 0) c.b++;
    c.nt = (c.len + tk - 1) / tk;
}
template <class G>
__device__ __forceinline__ void pa_next(const typename G::Args& a, const PaPlan& pl, PaCursor& c, int step) {
    if ((c.t += step) < c.nt) return;
    c.t = 0;
    if (++c.r < pl.units_row) return;
    c.r = 0;
    c.b++;
    pa_seek<G>(a, pl.tk, c);
}

// A wait that did not end at once: gives up after 2^31 SM cycles (about a
// second) and sets the error word; the warp's run then ends with that unit.
__device__ __noinline__ bool pa_wait_slow(uint64_t* bar, uint32_t parity, int* err) {
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity))
        if (clock64() - t0 > (1LL << 31)) {
            atomicOr(err, kPagedErrWait);
            return false;
        }
    return true;
}
__device__ __forceinline__ bool pa_wait(uint64_t* bar, uint32_t parity, int* err) {
    return mbar_try_wait(bar, parity) || pa_wait_slow(bar, parity, err);
}
// box of a map's tensor [page][slot][kv head][dim] -> shared memory (this CTA's)
__device__ __forceinline__ void pa_tensor_copy(uint32_t dst, const CUtensorMap* map, int h, int slot, int page,
                                               uint64_t* bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::"r"(dst),
        "l"(map), "r"(0), "r"(h), "r"(slot), "r"(page), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}

// What the warps of a CTA know of the line.
template <class G>
struct PaShared {
    long long scan[G::WARPS], ex[G::WARPS * 32], first[G::WARPS];
    PaCursor cur[G::WARPS];
};
struct PaRun {
    PaLine line;
    long long w0, u0, c0, c1;  // the CTA's first worker, this warp's first unit, the CTA's units
    bool worker, joint, whole, alone;
    int count, step;  // units of this warp, and from one to the next
    PaCursor cur;
    long long item0;  // first unit of the item that the run starts in
};
// Where this warp's run starts; rows of sequences without keys are zeroed here. All threads of the CTA.
template <class G>
__device__ __forceinline__ PaRun pa_start(const typename G::Args& a, const PaPlan& pl, PaShared<G>& sh, int hd) {
    constexpr int TK = G::TK, WARPS = G::WARPS;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = a.kv.num_seqs;
    const int team = pa_team<G>(pl), mate = warp / team;  // this warp's team
    PaRun run;
    // where the units of each sequence lie in the line
    const int per = (B + WARPS * 32 - 1) / (WARPS * 32);
    const int bs = min(B, tid * per), be = min(B, bs + per);
    long long mine = 0;
    bool none = false;  // one of this CTA's share of sequences has no key
    for (int b = bs; b < be; b++) {
        const int len = G::len(a, b);
        mine += (len + TK - 1) / TK;
        none |= len == 0 && b % gridDim.x == blockIdx.x;
    }
    mine *= pl.units_row;
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    if (lane == 31) sh.scan[warp] = incl;
    if (__syncthreads_or(none))  // rows of zeros
        for (int b = blockIdx.x; b < B; b += gridDim.x)
            if (G::len(a, b) == 0)
                for (int e = tid; e < a.H * hd; e += WARPS * 32) a.out[(size_t)b * a.ldo + e] = 0.0f;
    long long U = 0, ex = incl - mine;
    for (int w = 0; w < WARPS; w++) {
        if (w < warp) ex += sh.scan[w];
        U += sh.scan[w];
    }
    const PaLine line = run.line = pa_line(U, gridDim.x, WARPS / team, max(1, kPaFewWarps / team));
    const long long w0 = (long long)blockIdx.x * line.per_cta;
    sh.ex[tid] = ex;
    __syncthreads();
    {
        // where its run starts (the last thread's segment that starts at or before it)
        const long long u = line.start(w0 + mate);
        if (warp == mate * team && mate < line.per_cta && u < U) {
            int lo = 0;
#pragma unroll
            for (int i = 1 << (31 - __builtin_clz(WARPS * 32)); i > 0; i >>= 1)
                if (lo + i < WARPS * 32 && sh.ex[lo + i] <= u) lo += i;
            long long at = sh.ex[lo];
            for (int b = min(B, lo * per); b < B; b++) {
                const int len = G::len(a, b), nt = (len + TK - 1) / TK;
                const long long n = (long long)nt * pl.units_row;
                if (u < at + n) {
                    const long long k = u - at;
                    const int r = k >> 31 ? (int)(k / nt) : (int)k / nt, t0 = (int)(k - (long long)r * nt);
                    sh.cur[mate] = PaCursor{b, r, t0, nt, len};
                    sh.first[mate] = u - t0;  // first unit of the item that the run starts in
                    break;
                }
                at += n;
            }
        }
    }
    __syncthreads();

    run.worker = mate < line.per_cta;
    run.w0 = w0;
    run.u0 = line.start(w0 + mate);
    run.c0 = line.start(w0);
    run.c1 = line.start(w0 + line.per_cta);
    // joint: every run of the CTA inside one item: its warps take units in turn (neighbours in memory at the same
    // time) and are joined at the end. whole: and they are all of it
    run.joint = run.whole = false;
    if (run.c1 > run.c0) {
        const long long first = sh.first[0], end = first + sh.cur[0].nt;
        run.joint = run.c1 <= end;
        run.whole = run.c0 == first && run.c1 == end;
    }
    run.count = run.worker ? (int)(line.start(w0 + mate + 1) - run.u0) : 0;
    run.step = run.joint ? line.per_cta : 1;
    run.alone = run.whole && run.c1 - run.c0 == 1;
    run.cur = PaCursor{0, 0, 0, 0, 0};
    run.item0 = 0;
    if (run.joint) {
        run.cur = sh.cur[0];
        run.cur.t += mate;
        const int units = (int)(run.c1 - run.c0);
        run.count = run.worker && mate < units ? (units - mate + run.step - 1) / run.step : 0;
    } else if (run.count > 0) {
        run.cur = sh.cur[mate];
        run.item0 = sh.first[mate];
    }
    return run;
}

// A warp's sums of an item: lane (g, t) holds of query rows 8 e + 2 t, + 1 the dims 16 d + 2 g, + 1, references and
// sums. finish: the item's rows of out; store: a part of them at p.
template <class G>
__device__ __forceinline__ void pa_finish(const typename G::Args& a, const PaPlan& pl, const PaWork& work,
                                          const PaCursor& c, int hd, const float (&o)[G::HDP / 16][G::E][4],
                                          const float (&ref)[G::E][2], const float (&l)[G::E][2]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, group = a.H / a.KV;
    const int r = pa_row<G>(pl, c), qb = r % pl.qblocks, kvh = r / pl.qblocks;
#pragma unroll
    for (int e = 0; e < G::E; e++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int row = qb * G::ROWS + 8 * e + 2 * t + j;
            if (8 * e + 2 * t + j >= G::ROWS || row >= group) continue;
            float* out = a.out + (size_t)c.b * a.ldo + (size_t)(kvh * group + row) * hd;
            const float inv = l[e][j] == 0.0f ? 0.0f : __fdiv_rn(1.0f, l[e][j]);
            if (G::STAT && work.stat && g == 0)
                work.stat[(size_t)c.b * a.H + kvh * group + row] = make_float2(ref[e][j], inv);
#pragma unroll
            for (int d = 0; d < G::HDP / 16; d++)
                if (16 * d + 2 * g < hd) {
                    out[16 * d + 2 * g] = o[d][e][j] * inv;
                    out[16 * d + 2 * g + 1] = o[d][e][2 + j] * inv;
                }
        }
}
template <class G>
__device__ __forceinline__ void pa_store(float* p, bool any, const float (&o)[G::HDP / 16][G::E][4],
                                         const float (&ref)[G::E][2], const float (&l)[G::E][2]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int e = 0; e < G::E; e++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int row = 8 * e + 2 * t + j;
            if (row >= G::ROWS) continue;
            if (any)
#pragma unroll
                for (int d = 0; d < G::HDP / 16; d++)
                    *reinterpret_cast<float2*>(p + row * G::HDP + 16 * d + 2 * g) = make_float2(o[d][e][j], o[d][e][2 + j]);
            if (g == 0)
                *reinterpret_cast<float2*>(p + G::ROWS * G::HDP + 2 * row) =
                    any ? make_float2(ref[e][j], l[e][j]) : make_float2(kPaLow, 0.0f);
        }
}

// One warp's sum of parts for RB query rows: every load of a part is in flight
// at once. Lane i holds dims 4 i .. 4 i + 3 of every 128, and (ref, l) of row i % RB.
template <class G>
struct PaSum {
    static constexpr int HDP = G::HDP, RB = HDP <= 128 && G::ROWS >= 8 ? 8 : 4, NV = (HDP + 127) / 128;
    float4 o[RB][NV];
    float ref, l;
    // parts i = first, first + step, ... < np at work slots slot(i), rows r0 .. r0 + rows - 1
    template <class F>
    __device__ __forceinline__ void add(const float* part, int r0, int rows, int np, int first, int step, F slot) {
        const int lane = threadIdx.x & 31;
        ref = kPaLow;
        l = 0.0f;
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll
            for (int d = 0; d < NV; d++) o[r][d] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int i = first; i < np; i += step) {
            const float* p = part + (size_t)slot(i) * G::PART;
            const float2 rl = *reinterpret_cast<const float2*>(p + G::ROWS * HDP + 2 * (r0 + (lane & (RB - 1))));
            float4 x[RB][NV];
#pragma unroll
            for (int r = 0; r < RB; r++)
#pragma unroll
                for (int d = 0; d < NV; d++)
                    x[r][d] = r < rows && 128 * d + 4 * lane < HDP
                                  ? *reinterpret_cast<const float4*>(p + (r0 + r) * HDP + 128 * d + 4 * lane)
                                  : make_float4(0.f, 0.f, 0.f, 0.f);
            const float nr = fmaxf(ref, rl.x), fa = ex2(ref - nr), fb = ex2(rl.x - nr);
            l = __fmaf_rn(l, fa, rl.y * fb);
            ref = nr;
#pragma unroll
            for (int r = 0; r < RB; r++) {
                const float ga = __shfl_sync(0xffffffffu, fa, r), gb = __shfl_sync(0xffffffffu, fb, r);
#pragma unroll
                for (int d = 0; d < NV; d++) {
                    o[r][d].x = __fmaf_rn(o[r][d].x, ga, x[r][d].x * gb);
                    o[r][d].y = __fmaf_rn(o[r][d].y, ga, x[r][d].y * gb);
                    o[r][d].z = __fmaf_rn(o[r][d].z, ga, x[r][d].z * gb);
                    o[r][d].w = __fmaf_rn(o[r][d].w, ga, x[r][d].w * gb);
                }
            }
        }
    }
    __device__ __forceinline__ void store(float* p, int r0, int rows) const {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll
            for (int d = 0; d < NV; d++)
                if (r < rows && 128 * d + 4 * lane < HDP)
                    *reinterpret_cast<float4*>(p + (r0 + r) * HDP + 128 * d + 4 * lane) = o[r][d];
        if (lane < rows) *reinterpret_cast<float2*>(p + G::ROWS * HDP + 2 * (r0 + lane)) = make_float2(ref, l);
    }
    __device__ __forceinline__ void finish(float* out, int rows, int hd, float2* stat) const {
        const int lane = threadIdx.x & 31;
        if (G::STAT && stat && lane < rows) stat[lane] = make_float2(ref, l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l));
#pragma unroll
        for (int r = 0; r < RB; r++) {
            const float lr = __shfl_sync(0xffffffffu, l, r), inv = lr == 0.0f ? 0.0f : __fdiv_rn(1.0f, lr);
#pragma unroll
            for (int d = 0; d < NV; d++) {
                const int e = 128 * d + 4 * lane;
                if (r >= rows || e >= hd) continue;
                float* to = out + (size_t)r * hd + e;
                to[0] = o[r][d].x * inv;
                to[1] = o[r][d].y * inv;
                to[2] = o[r][d].z * inv;
                to[3] = o[r][d].w * inv;
            }
        }
    }
};

// The parts of the items that a CTA's runs share are joined: inside the CTA where an item ends in it, by
// paged_join_kernel otherwise. All threads, their runs being over; o, ref, l: this warp's sums of a joint CTA, kept in
// registers, the rings (RING bytes a warp at sm) being free. tail: the run ended inside the item `cur`, which it started at
// unit item0.
template <class G>
__device__ __forceinline__ void pa_end(const typename G::Args& a, const PaPlan& pl, const PaWork& work,
                                       const PaShared<G>& sh, const PaRun& run, int count, const PaCursor& cur,
                                       long long item0, bool tail, unsigned char* sm, int hd,
                                       const float (&o)[G::HDP / 16][G::E][4], const float (&ref)[G::E][2],
                                       const float (&l)[G::E][2]) {
    constexpr int HDP = G::HDP, ROWS = G::ROWS, WARPS = G::WARPS;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = a.H / a.KV;
    const int team = pa_team<G>(pl), mate = warp / team, member = warp - mate * team;
    const PaLine& line = run.line;
    const long long w0 = run.w0, c0 = run.c0, c1 = run.c1;
    // an item's part of worker w and this member: its later part (0) or its first (1)
    auto slot_at = [&](long long w, int m, int first) { return (int)(w * team + m) * 2 + first; };
    // CTAs behind this one that hold parts of an item that ends at unit `end`
    auto later = [&](long long end) { return (int)(line.worker(end - 1) / line.per_cta) - (int)blockIdx.x; };
    if (!run.joint) {
        // the items that this CTA's runs share: the warp where one starts joins its parts (warp 0 those of the
        // item that came into the CTA), in place
        __syncthreads();
        if (c1 == c0) return;
        const long long first = sh.first[0], end0 = first + sh.cur[0].nt;
        for (int pass = mate == 0 ? 0 : 1; pass < 2; pass++) {
            const bool head = pass == 0;
            if (head ? first >= c0 : !tail) continue;
            const long long end = head ? end0 : item0 + cur.nt;
            const int own = slot_at(w0 + mate, member, head ? 0 : 1);
            int np = 1;
            while (mate + np < line.per_cta && line.start(w0 + mate + np) < end) np++;
            const PaCursor it = head ? sh.cur[0] : cur;
            const bool ends = !head && end <= c1;
            if (!head && !ends && lane == 0 && member == 0)
                work.tail[blockIdx.x] = PaTail{later(end), own, it.b, it.r, line.per_cta};
            if (np == 1) continue;
            const int r = pa_row<G>(pl, it), qb = r % pl.qblocks, kvh = r / pl.qblocks;
            auto slot_of = [&](int i) { return i == 0 ? own : slot_at(w0 + mate + i, member, 0); };
            for (int r0 = 0; r0 < ROWS && qb * ROWS + r0 < group; r0 += PaSum<G>::RB) {
                PaSum<G> sum;
                const int rows = min(PaSum<G>::RB, group - qb * ROWS - r0);
                sum.add(work.part, r0, rows, np, 0, 1, slot_of);
                if (ends)
                    sum.finish(a.out + (size_t)it.b * a.ldo + (size_t)(kvh * group + qb * ROWS + r0) * hd, rows, hd,
                               work.stat ? work.stat + (size_t)it.b * a.H + kvh * group + qb * ROWS + r0 : nullptr);
                else
                    sum.store(work.part + (size_t)own * G::PART, r0, rows);
            }
        }
        return;
    }
    if (run.alone) return;  // written

    const int begins = c0 == sh.first[0] ? 1 : 0;
    if (tid == 0 && !run.whole && begins)
        work.tail[blockIdx.x] = PaTail{later(sh.first[0] + sh.cur[0].nt), slot_at(w0, 0, 1), sh.cur[0].b, sh.cur[0].r, line.per_cta};
    if (G::TEAM && line.per_cta == 1 && !run.whole) {  // one worker: its sums are the CTA's part
        if (run.worker) pa_store<G>(work.part + (size_t)slot_at(w0, member, begins) * G::PART, true, o, ref, l);
        return;
    }
    // join the CTA's workers (their rings are free now)
    if (run.worker) pa_store<G>(reinterpret_cast<float*>(sm + warp * G::RING), count > 0, o, ref, l);
    __syncthreads();
    const PaCursor c = sh.cur[0];
    for (int i = tid; i < team * (ROWS * HDP / 4); i += WARPS * 32) {
        const int m = G::TEAM ? i / (ROWS * HDP / 4) : 0, k = i - m * (ROWS * HDP / 4);
        const int row = k / (HDP / 4), d = k % (HDP / 4) * 4, r = c.r * team + m, qb = r % pl.qblocks, kvh = r / pl.qblocks;
        float* part = work.part + (size_t)slot_at(w0, m, begins) * G::PART;
        float M = kPaLow, L = 0.0f;
        float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int w = 0; w < line.per_cta; w++)
            M = fmaxf(M, reinterpret_cast<const float*>(sm + (w * team + m) * G::RING)[ROWS * HDP + 2 * row]);
#pragma unroll 1
        for (int w = 0; w < line.per_cta; w++) {
            const float* wb = reinterpret_cast<const float*>(sm + (w * team + m) * G::RING);
            const float wr = wb[ROWS * HDP + 2 * row], wl = wb[ROWS * HDP + 2 * row + 1];
            if (wl == 0.0f) continue;  // no key (a warp without units left no o)
            const float f = ex2(wr - M);
            const float4 x = *reinterpret_cast<const float4*>(wb + row * HDP + d);
            L = __fmaf_rn(f, wl, L);
            O = make_float4(__fmaf_rn(f, x.x, O.x), __fmaf_rn(f, x.y, O.y), __fmaf_rn(f, x.z, O.z), __fmaf_rn(f, x.w, O.w));
        }
        if (run.whole) {
            if (qb * ROWS + row < group && d < hd) {
                float* out = a.out + (size_t)c.b * a.ldo + (size_t)(kvh * group + qb * ROWS + row) * hd + d;
                const float inv = L == 0.0f ? 0.0f : __fdiv_rn(1.0f, L);
                if (G::STAT && work.stat && d == 0)
                    work.stat[(size_t)c.b * a.H + kvh * group + qb * ROWS + row] = make_float2(M, inv);
                out[0] = O.x * inv;
                out[1] = O.y * inv;
                out[2] = O.z * inv;
                out[3] = O.w * inv;
            }
        } else {
            *reinterpret_cast<float4*>(part + row * HDP + d) = O;
            if (d == 0) *reinterpret_cast<float2*>(part + ROWS * HDP + 2 * row) = make_float2(M, L);
        }
    }
}

// The items that start in one CTA of the kernel above and end in a later one:
// a CTA each. Warp w adds parts w, w + 8, ..., then the warps' sums are joined
// in shared memory.
constexpr int kPaJoinWarps = 8;
template <class G>
__global__ void __launch_bounds__(kPaJoinWarps * 32)
    paged_join_kernel(typename G::Args a, PaPlan pl, PaWork work) {
    using Sum = PaSum<G>;
    constexpr int HDP = G::HDP, ROWS = G::ROWS, NV = Sum::NV, RB = Sum::RB;
    __shared__ __align__(16) float s_o[kPaJoinWarps][RB][HDP];
    __shared__ float2 s_rl[kPaJoinWarps][RB];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = a.H / a.KV, hd = a.hd;
    griddep_wait();
    const PaTail tail = work.tail[blockIdx.x];
    if (tail.ctas == 0) return;
    const int np = tail.ctas + 1, qb = tail.r % pl.qblocks, kvh = tail.r / pl.qblocks;
    auto slot_of = [&](int i) { return i == 0 ? tail.slot : ((int)blockIdx.x + i) * tail.per_cta * 2; };
    for (int r0 = 0; r0 < ROWS && qb * ROWS + r0 < group; r0 += RB) {
        const int rows = min(RB, group - qb * ROWS - r0);
        Sum sum;
        sum.add(work.part, r0, rows, np, warp, kPaJoinWarps, slot_of);
        if (r0) __syncthreads();  // the last row block's sums are read
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll
            for (int d = 0; d < NV; d++)
                if (128 * d + 4 * lane < HDP) *reinterpret_cast<float4*>(&s_o[warp][r][128 * d + 4 * lane]) = sum.o[r][d];
        if (lane < RB) s_rl[warp][lane] = make_float2(sum.ref, sum.l);
        __syncthreads();
        const int used = min(np, kPaJoinWarps);
        for (int i = tid; i < rows * HDP; i += kPaJoinWarps * 32) {
            const int r = i / HDP, d = i % HDP;
            float M = kPaLow, L = 0.0f, O = 0.0f;
            for (int w = 0; w < used; w++) M = fmaxf(M, s_rl[w][r].x);
            for (int w = 0; w < used; w++) {
                const float f = ex2(s_rl[w][r].x - M);
                L = __fmaf_rn(f, s_rl[w][r].y, L);
                O = __fmaf_rn(f, s_o[w][r][d], O);
            }
            if (d < hd)
                a.out[(size_t)tail.b * a.ldo + (size_t)(kvh * group + qb * ROWS + r0 + r) * hd + d] =
                    L == 0.0f ? 0.0f : __fdiv_rn(O, L);
        }
    }
}

// The same for teams, whose items go through more CTAs: blockIdx.y takes pa_wide_rows query rows of a team's rows.
// One row at a time: the threads find the reference and the parts' factors, then each adds four dims over its share of the
// parts, kPaWideLoads of them in flight, and the shares are added in shared memory. Small CTAs, as most find nothing to
// join. (148 parts of 8 heads' 4 rows of 128: 8 us, about 10 with 512 threads for the 4 rows at once.)
constexpr int kPaWideThreads = 128, kPaWideLoads = 16, kPaMaxCtas = 256;
template <class G>
__host__ __device__ constexpr int pa_wide_rows(int team) {
    return G::ROWS * team > 32 ? (G::ROWS * team + 31) / 32 : 1;
}
template <class G>
__global__ void __launch_bounds__(kPaWideThreads) paged_join_wide_kernel(typename G::Args a, PaPlan pl, PaWork work) {
    constexpr int HDP = G::HDP, ROWS = G::ROWS, COLS = HDP / 4, SIDE = kPaWideThreads / COLS, WARPS = kPaWideThreads / 32;
    constexpr int REFS = kPaMaxCtas / kPaWideThreads;
    static_assert(COLS <= kPaWideThreads, "a row's columns fit the threads");
    __shared__ float s_f[kPaMaxCtas], s_m[WARPS], s_l[WARPS];
    __shared__ __align__(16) float4 s_o[kPaWideThreads];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = a.H / a.KV, hd = a.hd;
    if (G::STAT) griddep_launch();
    griddep_wait();
    const PaTail tail = work.tail[blockIdx.x];
    if (tail.ctas == 0) return;
    const int team = pa_team<G>(pl), np = tail.ctas + 1, each = pa_wide_rows<G>(team);
    for (int k = 0; k < each; k++) {
        const int at = blockIdx.y * each + k, member = at / ROWS, row = at - member * ROWS;
        const int item = tail.r * team + member, qb = item % pl.qblocks, kvh = item / pl.qblocks;
        if (member >= team || qb * ROWS + row >= group) continue;  // the whole CTA
        const int h = kvh * group + qb * ROWS + row;
        auto part = [&](int i) {
            return work.part + (size_t)((i == 0 ? tail.slot : ((int)blockIdx.x + i) * tail.per_cta * team * 2) + member * 2) * G::PART;
        };
        float2 rl[REFS];
        float M = kPaLow, L = 0.0f;
#pragma unroll
        for (int i = 0; i < REFS; i++) {
            const int n = tid + kPaWideThreads * i;
            rl[i] = n < np ? *reinterpret_cast<const float2*>(part(n) + ROWS * HDP + 2 * row) : make_float2(kPaLow, 0.0f);
            M = fmaxf(M, rl[i].x);
        }
        // the first loads of the rows need no factors
        const int col = tid % COLS, side = tid / COLS, d = 4 * col;
        float4 x[kPaWideLoads];
        auto load = [&](int i0) {
#pragma unroll
            for (int i = 0; i < kPaWideLoads; i++)
                x[i] = side < SIDE && i0 + SIDE * i < np ? *reinterpret_cast<const float4*>(part(i0 + SIDE * i) + row * HDP + d)
                                                        : make_float4(0.f, 0.f, 0.f, 0.f);
        };
        load(side);
        M = warp_max(M);
        if (lane == 0) s_m[warp] = M;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WARPS; w++) M = fmaxf(M, s_m[w]);
#pragma unroll
        for (int i = 0; i < REFS; i++) {
            const float f = ex2(rl[i].x - M);
            s_f[tid + kPaWideThreads * i] = f;
            L = __fmaf_rn(rl[i].y, f, L);
        }
        L = warp_sum(L);
        if (lane == 0) s_l[warp] = L;
        __syncthreads();
        L = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) L += s_l[w];
        const float inv = L == 0.0f ? 0.0f : __fdiv_rn(1.0f, L);
        if (G::STAT && work.stat && tid == 0) work.stat[(size_t)tail.b * a.H + h] = make_float2(M, inv);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = side; i0 < np; i0 += SIDE * kPaWideLoads) {
            if (i0 != side) load(i0);
#pragma unroll
            for (int i = 0; i < kPaWideLoads; i++) {
                const float f = i0 + SIDE * i < np ? s_f[i0 + SIDE * i] : 0.0f;
                o = make_float4(__fmaf_rn(x[i].x, f, o.x), __fmaf_rn(x[i].y, f, o.y), __fmaf_rn(x[i].z, f, o.z),
                                __fmaf_rn(x[i].w, f, o.w));
            }
        }
        s_o[tid] = o;
        __syncthreads();
        if (side == 0 && d < hd) {
#pragma unroll
            for (int w = 1; w < SIDE; w++) {
                const float4 y = s_o[w * COLS + tid];
                o = make_float4(o.x + y.x, o.y + y.y, o.z + y.z, o.w + y.w);
            }
            float* to = a.out + (size_t)tail.b * a.ldo + (size_t)h * hd + d;
            to[0] = o.x * inv;
            to[1] = o.y * inv;
            to[2] = o.z * inv;
            to[3] = o.w * inv;
        }
        __syncthreads();  // the next row takes the shared arrays
    }
}

}  // namespace

}  // namespace jyc
