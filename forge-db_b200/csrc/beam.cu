// beam.cu -- one step of a beam search: the best continuations over beams and
// columns, and states that follow the beams they were taken from.
//
//   l_bj = scale x_bj - log sum_j exp(scale x_bj)   (or scale x_bj)
//   the `width` largest beam_b + l_bj, equal ones by beam, then column
//
// Scores are compared in 64 bits, as a 32-bit sum of two of them would make equal
// what is not.
#include <climits>
#include <cmath>

#include "softmax_rows.cuh"

namespace fdb {
namespace beam {

using sr::Carve;
using sr::hi_of;
using sr::lo_of;
using sr::packf;
using sr::to_f32;
using sr::up;

// What a chain's columns are read from.
struct Select {
    const void* x;
    int beams, n, width;
    size_t ld_group, ld_beam;
    double scale;
    int normalise;
    const int64_t* ids;
    size_t ld_ids;
    const uint32_t* allowed;
    size_t ld_allowed;
    const float* beam_scores;
    const uint8_t* ended;
    int64_t end_id;
    float* out_scores;
    int64_t *out_parents, *out_ids;
    uint8_t* out_ended;
};

// A column's x, -inf if it takes no part.
template <typename T>
__device__ __forceinline__ float column(const Select& p, int g, int b, int j) {
    const size_t row = (size_t)g * p.beams + b;
    // (all loads first)
    const float x = to_f32<T>(static_cast<const T*>(p.x)[(size_t)g * p.ld_group + (size_t)b * p.ld_beam + j]);
    const int64_t id = p.ids ? p.ids[row * p.ld_ids + j] : 0;
    const uint32_t w = p.allowed ? p.allowed[row * p.ld_allowed + (j >> 5)] : 0xffffffffu;
    return id < 0 || !(w >> (j & 31) & 1u) ? -INFINITY : x;
}
__device__ __forceinline__ bool over(const Select& p, int g, int b) {
    return p.ended && p.ended[(size_t)g * p.beams + b];
}
// A chain that is not there: whatever its columns hold.
__device__ __forceinline__ bool absent(const Select& p, int g, int b) {
    return p.beam_scores[(size_t)g * p.beams + b] == -INFINITY;
}

// ---------------------------------------------------------------------------
// order-preserving images of numbers (of -0 and 0 the same)
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t ordered(float f) {
    const uint32_t u = __float_as_uint(f + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint64_t ordered64(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double unordered64(uint64_t u) {
    return __longlong_as_double((long long)(u >> 63 ? u & 0x7fffffffffffffffull : ~u));
}

// ---------------------------------------------------------------------------
// scanning the chains' columns
// ---------------------------------------------------------------------------
// A block takes a part of a chain's columns, a tile of TH * U loads of 16 bytes at a
// time, and leaves their sum of exponentials and the `width` best.  The pass over the
// columns only adds up and keeps each thread's largest of a span of tiles, without a
// barrier.  The best are found from those maxima afterwards: of the threads' largest the
// width-th (or, for 16 at most, the least of the largest of G >= width groups of threads) is
// reached by at least `width` columns and by hardly more; only the maxima that reach it
// are looked behind, by reading their columns again.
// Sums are taken relative to a thread's own largest score so far (raised only when it
// is exceeded by 2^8), a tile's terms in f32 and those in 64 bits.
// 64 x 8 x 131072 columns, width 8: f32 48 us (5.5 TB/s, where a copy has 6.4), bf16 30
// (4.5 TB/s): a block's start and end, some 4 us without loads, and one exponential a
// column (40 % of their unit's rate).  Looking for the best column by column, as they
// come, took 74 us; a block for each search's last to end, with the finish, 46.  With
// filters or ids the columns pass through registers, one tile ahead, and each is tested:
// the same chains with a filter each take 94 and 57 us.
constexpr int TH = 256;               // threads
constexpr int U = 4;                  // loads of a thread in a tile
constexpr int SPAN = 2;               // tiles whose largest is kept together
constexpr int SPANS = 16;             // of a block
constexpr int RING = 2;               // tiles on their way
constexpr int GROUPS = 1024;          // maxima looked behind at once
constexpr int MAXW = FDB_MAX_BEAMS;
constexpr float RAISE = 8.0f;

template <typename T>
struct Vec;  // 16 bytes of columns
template <>
struct Vec<float> {
    static constexpr int N = 4;
    static constexpr uint32_t NONE = 0xff800000u;  // -inf, in every element of a word
    // the largest (NaN if one is) of U vectors
    static __device__ __forceinline__ float most(const uint4 (&r)[U]) {
        float m = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(__uint_as_float(r[u].x)));
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(__uint_as_float(r[u].y)));
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(__uint_as_float(r[u].z)));
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(__uint_as_float(r[u].w)));
        }
        return m;
    }
    static __device__ __forceinline__ float2 pair(const uint4& r, int i) {
        return i ? make_float2(__uint_as_float(r.z), __uint_as_float(r.w))
                 : make_float2(__uint_as_float(r.x), __uint_as_float(r.y));
    }
};
template <>
struct Vec<__half> {
    static constexpr int N = 8;
    static constexpr uint32_t NONE = 0xfc00fc00u;
    static __device__ __forceinline__ float most(const uint4 (&r)[U]) {
        const __half2* h = reinterpret_cast<const __half2*>(r);
        __half2 m = h[0];
#pragma unroll
        for (int i = 1; i < 4 * U; ++i) m = __hmax2_nan(m, h[i]);
        const float2 f = __half22float2(m);
        float v;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(f.x), "f"(f.y));
        return v;
    }
    static __device__ __forceinline__ float2 pair(const uint4& r, int i) {
        return __half22float2(reinterpret_cast<const __half2*>(&r)[i]);
    }
};
template <>
struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static constexpr uint32_t NONE = 0xff80ff80u;
    static __device__ __forceinline__ float most(const uint4 (&r)[U]) {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(r);
        __nv_bfloat162 m = h[0];
#pragma unroll
        for (int i = 1; i < 4 * U; ++i) m = __hmax2_nan(m, h[i]);
        const float2 f = __bfloat1622float2(m);
        float v;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(f.x), "f"(f.y));
        return v;
    }
    static __device__ __forceinline__ float2 pair(const uint4& r, int i) {
        const uint32_t w = reinterpret_cast<const uint32_t*>(&r)[i];
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
};

// What a block leaves: sum of 2^((x - m) s), its `count` best columns in order.
struct Part {
    double sum;
    float m;
    int count;  // -1: a column is NaN or +inf
};
struct Scan {
    Part* part;       // [chains][splits]
    uint64_t* best;   // [chains][splits][width]: ordered(x) << 32 | ~column
    int splits;
    float s;          // scale log2(e)
    float slack;      // see finish_kernel
};

// Vector v of a chain whose first column is `skip` columns into vector 0; columns
// outside of it, or that take no part, as -inf.
template <typename T, bool GATE>
__device__ __forceinline__ uint4 load_vec(const Select& p, const T* x, int skip, size_t row, int v,
                                          int v1) {
    constexpr int N = Vec<T>::N;
    uint4 r = make_uint4(Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE);
    if (v >= v1) return r;
    const int j0 = v * N - skip;
    if (j0 >= 0 && j0 <= p.n - N) {
        r = __ldcs(reinterpret_cast<const uint4*>(x + j0));
    } else {
        T* e = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (j0 + i >= 0 && j0 + i < p.n) e[i] = x[j0 + i];
    }
    if (GATE) {
        uint32_t keep = (1u << N) - 1;
        if (p.allowed) {
            const uint32_t* al = p.allowed + row * p.ld_allowed;
            const int lo = max(j0, 0), w = lo >> 5;
            uint64_t bits = __ldg(al + w);
            if (w + 1 < (p.n + 31) >> 5) bits |= (uint64_t)__ldg(al + w + 1) << 32;
            keep &= (uint32_t)(bits >> (lo & 31)) << (lo - j0);
        }
        if (p.ids) {
            const int64_t* id = p.ids + row * p.ld_ids;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (j0 + i >= 0 && j0 + i < p.n && __ldg(id + j0 + i) < 0) keep &= ~(1u << i);
        }
        const uint4 none = make_uint4(Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE);
        T* e = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (!(keep >> i & 1u)) e[i] = reinterpret_cast<const T*>(&none)[i];
    }
    return r;
}

// The width-th largest of the threads' values (images of `ordered`): each warp sorts its
// own into `sorted` [TH], a thread looks for its place among the eight.  (Comparing each
// with all took 6 us of a scan's end.)  *bound is all ones, behind a barrier.
__device__ __forceinline__ uint32_t width_th(uint32_t v, int width, uint32_t* sorted,
                                             uint32_t* bound) {
    const int tid = threadIdx.x, lane = tid & 31;
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j; j >>= 1) {
            const uint32_t o = __shfl_xor_sync(0xffffffffu, v, j);
            v = ((lane & k) == 0) == ((lane & j) == 0) ? max(v, o) : min(v, o);
        }
    sorted[tid] = v;  // (falling)
    __syncthreads();
    int above = 0;
#pragma unroll
    for (int w = 0; w < TH / 32; ++w) {
        int at = 0;  // (how many of the warp's are larger)
#pragma unroll
        for (int step = 16; step; step >>= 1)
            if (sorted[w * 32 + at + step - 1] > v) at += step;
        if (sorted[w * 32 + at] > v) ++at;
        above += at;
    }
    const uint32_t least = __reduce_min_sync(0xffffffffu, above < width ? v : ~0u);
    if (lane == 0) atomicMin(bound, least);
    __syncthreads();
    return *bound;
}

// ---- the best of what lies in shared memory ----
constexpr int LIMIT = 256;              // keys that are put in order at once
constexpr int ASIDE = 512;
struct Best {
    uint64_t* buf;                      // [LIMIT + TH * columns of a vector]
    alignas(16) uint64_t aside[ASIDE];  // (read four floats at a time, too)
    uint64_t out[MAXW], least;
    int count, total;
};
// Leaves the `width` best of s.count keys, which all differ, in order at buf's front
// and returns how many they are.  Ranks are counted; of more than TH keys only
// those that reach the width-th largest of TH maxima are ranked.  Called by all
// threads, after a barrier.
__device__ __forceinline__ int keep_best(Best& s, int width) {
    const int tid = threadIdx.x;
    const uint64_t* from = s.buf;
    int n = s.count;
    if (n > TH) {
        uint64_t m = 0;
        for (int i = tid; i < n; i += TH) m = max(m, s.buf[i]);
        s.aside[tid] = m;
        if (tid == 0) s.total = 0;
        __syncthreads();
        int rank = 0;
#pragma unroll 8
        for (int i = 0; i < TH; ++i) rank += s.aside[i] > m;
        if (rank == width - 1) s.least = m;
        __syncthreads();
        const uint64_t least = s.least;
        for (int i = tid; i < n; i += TH) {
            const uint64_t v = s.buf[i];
            if (v < least) continue;
            const int at = atomicAdd(&s.total, 1);
            if (at < ASIDE) s.aside[at] = v;
        }
        __syncthreads();
        if (s.total <= ASIDE) n = s.total, from = s.aside;
    }
    for (int i = tid; i < n; i += TH) {
        const uint64_t v = from[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) rank += from[j] > v;
        if (rank < width) s.out[rank] = v;
    }
    __syncthreads();
    n = min(n, width);
    for (int i = tid; i < n; i += TH) s.buf[i] = s.out[i];
    if (tid == 0) s.count = n;
    __syncthreads();
    return n;
}

// (the copies in flight are done with when the best are looked for)
template <typename T>
struct ScanShared {
    union {
        uint4 ring[RING][U][TH];
        struct {
            uint64_t buf[LIMIT + TH * Vec<T>::N];
            Best s;
            int list[GROUPS];
        } e;
    };
    float top[SPANS][TH];  // a thread's largest of each span
    float warp_min[TH / 32], warp_m[TH / 32];
    uint32_t bound;
    int groups;
    double warp_sum[TH / 32];
};
// What a thread's exponents are relative to: 2^(x s - reference).  Below the range
// where x s stays finite its terms are 0 (finish_kernel takes such sums again).
__device__ __forceinline__ float reference(float m, float s) { return fmaxf(m * s, -1e30f); }
template <typename T, bool NORM, bool GATE>
__device__ __forceinline__ void scan_part(const Select& p, const Scan& c, ScanShared<T>& sh,
                                          size_t row, int sp, int g, int b) {
    constexpr int N = Vec<T>::N, STEP = TH * U;
    Best& s = sh.e.s;
    uint64_t* buf = sh.e.buf;
    const int tid = threadIdx.x;
    const T* x = static_cast<const T*>(p.x) + (size_t)g * p.ld_group + (size_t)b * p.ld_beam;
    const int skip = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    const long long nv = ((long long)p.n + skip + N - 1) / N;
    const int v0 = (int)(nv * sp / c.splits), v1 = (int)(nv * (sp + 1) / c.splits);
    const int tiles = (v1 - v0 + STEP - 1) / STEP, spans = (tiles + SPAN - 1) / SPAN;
    if (tid == 0) sh.groups = 0, sh.bound = ~0u;

    // ---- sums, and the largest of each thread's columns of a tile ----
    // Without gates a thread's loads go through its own places of a ring in shared
    // memory, RING tiles ahead; else through registers, one ahead.
    float m = 0.0f, ref = 0.0f, most = -INFINITY, span = -INFINITY;
    double sum = 0.0;
    bool started = false;
    uint4 next[GATE ? U : 1];
    const uint4* vecs = reinterpret_cast<const uint4*>(x - skip);
    // (tiles of whole vectors, in the row from end to end)
    const int whole0 = skip ? 1 : 0, whole1 = min(v1, (int)(((long long)p.n + skip) / N));
    auto whole = [&](int t) { return v0 + t * STEP >= whole0 && v0 + (t + 1) * STEP <= whole1; };
    const uint4* mine = vecs + v0 + tid;
    const uint32_t places = (uint32_t)__cvta_generic_to_shared(&sh.ring[0][0][tid]);
    auto fetch = [&](int t) {
        if (GATE) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                next[u * GATE] = load_vec<T, GATE>(p, x, skip, row, v0 + t * STEP + u * TH + tid, v1);
        } else if (whole(t)) {
            const uint4* src = mine + t * STEP;
#pragma unroll
            for (int u = 0; u < U; ++u)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                                 places + (uint32_t)((t % RING * U + u) * TH * 16)),
                             "l"(src + u * TH)
                             : "memory");
        }  // (others are read when it is their turn)
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int t = 0; t < (GATE ? 1 : RING); ++t)
        if (t < tiles) fetch(t);
        else asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll 1
    for (int t = 0; t < tiles; ++t) {
        uint4 r[U];
        if (GATE) {
#pragma unroll
            for (int u = 0; u < U; ++u) r[u] = next[u * GATE];
            if (t + 1 < tiles) fetch(t + 1);
        } else {
            asm volatile("cp.async.wait_group %0;" ::"n"(RING - 1) : "memory");
            if (whole(t)) {
#pragma unroll
                for (int u = 0; u < U; ++u) r[u] = sh.ring[t % RING][u][tid];
            } else {
#pragma unroll
                for (int u = 0; u < U; ++u)
                    r[u] = load_vec<T, false>(p, x, skip, row, v0 + t * STEP + u * TH + tid, v1);
            }
            if (t + RING < tiles) fetch(t + RING);
            else asm volatile("cp.async.commit_group;" ::: "memory");
        }
        const float top = Vec<T>::most(r);
        if (t % SPAN) asm("max.NaN.f32 %0, %0, %1;" : "+f"(span) : "f"(top));
        else span = top;
        if (t % SPAN == SPAN - 1 || t + 1 == tiles) {
            sh.top[t / SPAN][tid] = span;
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(span));
        }
        if (NORM) {
            if (top > -INFINITY && (!started || (top - m) * c.s > RAISE)) {
                const float to = reference(top, c.s);
                if (started) sum *= (double)sr::ex2(ref - to);
                m = top;
                ref = to;
                started = true;
            }
            const uint64_t c2 = packf(-ref, -ref), s2 = packf(c.s, c.s);
            uint64_t acc[2] = {0, 0};
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < N / 2; ++i) {
                    const float2 f = Vec<T>::pair(r[u], i);
                    const uint64_t t2 = tc::fma2(packf(f.x, f.y), s2, c2);
                    acc[i & 1] = tc::add2(acc[i & 1], packf(sr::ex2(lo_of(t2)), sr::ex2(hi_of(t2))));
                }
            const uint64_t both = tc::add2(acc[0], acc[1]);
            sum += (double)(lo_of(both) + hi_of(both));
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    // (finish_kernel's blocks may take their places: they wait for this grid's results)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // ---- a bound that at least `width` columns reach; the sums ----
    float bound = most, M = started ? m : -INFINITY;
    const int group = p.width <= 8 ? 32 : 16;  // (of threads, for 8 or 16 groups)
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const float v = __shfl_xor_sync(0xffffffffu, bound, o);
        bound = o < group ? fmaxf(bound, v) : fminf(bound, v);
        if (NORM) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    }
    if ((tid & 31) == 0) sh.warp_min[tid >> 5] = bound, sh.warp_m[tid >> 5] = M;
    const bool bad = __syncthreads_or(!(most < INFINITY));
    if (tid == 0) s.count = 0, s.buf = buf;
    float tau = sh.warp_min[0];
#pragma unroll
    for (int i = 1; i < TH / 32; ++i) tau = fminf(tau, sh.warp_min[i]);
    // (or a group has no column, and all columns would reach it)
    if (p.width > 16 || tau == -INFINITY)
        tau = unordered(width_th(ordered(most), p.width, reinterpret_cast<uint32_t*>(s.aside),
                                 &sh.bound));
    if (NORM) {
#pragma unroll
        for (int i = 0; i < TH / 32; ++i) M = fmaxf(M, sh.warp_m[i]);
        // (what rounding the reference moved, and the distance of the block's)
        if (sum > 0.0)
            sum *= (double)sr::ex2((float)((double)ref - (double)m * c.s)) *
                   (double)sr::ex2((m - M) * c.s);
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if ((tid & 31) == 0) sh.warp_sum[tid >> 5] = sum;
    }
    // ---- the maxima that reach it, and the columns behind them ----
    if (bad) {
        if (tid == 0) c.part[blockIdx.x] = Part{0.0, 0.0f, -1};
        return;
    }
    if (most > -INFINITY && most >= tau) {
        for (int t = 0; t < spans; ++t) {
            const float top = sh.top[t][tid];
            if (top > -INFINITY && top >= tau) {
                const int to = atomicAdd(&sh.groups, 1);
                if (to < GROUPS) sh.e.list[to] = t * TH + tid;
            }
        }
    }
    __syncthreads();
    const int groups = sh.groups;
    auto enter = [&](const uint4& v, int first, bool reach, int room) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const float2 f = Vec<T>::pair(v, i);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float y = h ? f.y : f.x;
                if (!(y > -INFINITY) || !(reach ? y >= tau : y > tau)) continue;
                const int to = atomicAdd(&s.count, 1);
                if (to < room) buf[to] = (uint64_t)ordered(y) << 32 | (uint32_t)~(first + 2 * i + h);
            }
        }
    };
    constexpr int ROOM = LIMIT + TH * N;
    bool all = groups > GROUPS;
    if (!all) {
        for (int k = tid; k < groups * (SPAN * U); k += TH) {
            const int e = sh.e.list[k / (SPAN * U)];
            const int at = v0 + (e / TH * (SPAN * U) + k % (SPAN * U)) * TH + e % TH;
            enter(load_vec<T, GATE>(p, x, skip, row, at, v1), at * N - skip, true, ROOM);
        }
        __syncthreads();
        all = s.count > ROOM;
    }
    if (all) {
        // too many columns are as good: span by span, the best kept at any time.  (A
        // column that equals the width-th and lies further on is not better.)
        __syncthreads();
        if (tid == 0) s.count = 0;
        __syncthreads();
        bool reach = true;
        for (int t = 0; t < spans; ++t) {
            const float top = sh.top[t][tid];
            const bool hit = top > -INFINITY && (reach ? top >= tau : top > tau);
            if (!__syncthreads_or(hit)) continue;
#pragma unroll 1
            for (int u = 0; u < SPAN * U; ++u) {
                const int at = v0 + (t * (SPAN * U) + u) * TH + tid;
                if (hit) enter(load_vec<T, GATE>(p, x, skip, row, at, v1), at * N - skip, reach, ROOM);
                __syncthreads();
                const bool full = s.count >= LIMIT;
                __syncthreads();
                if (full && keep_best(s, p.width) == p.width) {
                    tau = unordered((uint32_t)(buf[p.width - 1] >> 32));
                    reach = false;
                }
            }
        }
    }
    __syncthreads();
    uint64_t* out = c.best + (size_t)blockIdx.x * p.width;
    const int count = s.count, have = min(count, p.width);
    if (count <= TH) {
        if (tid < count) {
            const uint64_t v = buf[tid];
            int rank = 0;
#pragma unroll 4
            for (int i = 0; i < count; ++i) rank += buf[i] > v;
            if (rank < p.width) out[rank] = v;
        }
    } else {
        keep_best(s, p.width);
        for (int i = tid; i < have; i += TH) out[i] = buf[i];
    }
    if (tid == 0) {
        double v = 0.0;
        if (NORM)
            for (int i = 0; i < TH / 32; ++i) v += sh.warp_sum[i];
        c.part[blockIdx.x] = Part{v, M, have};
    }
}

// ---------------------------------------------------------------------------
// the best of all chains
// ---------------------------------------------------------------------------
constexpr int CAP = 2048, ROUND = 1024;
enum { LIVE = 0, OVER = 1, ABSENT = 2 };
struct Choice {
    uint64_t score[CAP], at[CAP];       // ordered64; chain << 32 | column
    uint64_t near_score[ASIDE], near_at[ASIDE];
    float set[TH];
    uint32_t bound;
    double out_score[MAXW];
    uint64_t out_at[MAXW];
    int count, total, have;
};
__device__ __forceinline__ void add(Choice& s, double v, int b, int j) {
    const int to = atomicAdd(&s.count, 1);
    s.score[to] = ordered64(v);
    s.at[to] = (uint64_t)b << 32 | (uint32_t)j;
}
// The width-th largest of s.set[0, n), n <= TH (-inf if there are fewer).  Called by all
// threads, after a barrier; s.bound is all ones.
__device__ __forceinline__ float bound_of(Choice& s, int n, int width) {
    if (n < width) return -INFINITY;
    const int tid = threadIdx.x;
    if (n <= 32) {  // (a few comparisons are done sooner)
        if (tid < n) {
            const float v = s.set[tid];
            int above = 0;
#pragma unroll 8
            for (int i = 0; i < n; ++i) above += s.set[i] > v;
            if (above < width) atomicMin(&s.bound, ordered(v));
        }
        __syncthreads();
        return unordered(s.bound);
    }
    // (what is sorted takes its places)
    return unordered(width_th(tid < n ? ordered(s.set[tid]) : 0u, width,
                              reinterpret_cast<uint32_t*>(s.set), &s.bound));
}
// Of the candidates that the threads hold (-inf: none) those not `slack` below the
// width-th of s.set[0, n) are added.
constexpr int HELD = 4;
template <int H>
__device__ __forceinline__ void pick(Choice& s, const double (&v)[H], const int (&b)[H],
                                     const int (&j)[H], int n, int width, double slack) {
    __syncthreads();
    const double least = (double)bound_of(s, n, width) - slack;
#pragma unroll
    for (int h = 0; h < H; ++h)
        if (v[h] > -INFINITY && v[h] >= least) add(s, v[h], b[h], j[h]);
    __syncthreads();
}
// The candidates whose scores are not `slack` below the width-th, those in front
// ranked into out_*.  Returns them: [0, n) of `score` and `at`.  Called by all
// threads, after a barrier.
struct Ranked {
    const uint64_t *score, *at;
    int n;
};
__device__ __forceinline__ Ranked rank_all(Choice& s, int width, double slack) {
    const int tid = threadIdx.x;
    Ranked r{s.score, s.at, s.count};
    if (r.n > TH) {
        float m = -INFINITY;
        for (int i = tid; i < r.n; i += TH) m = fmaxf(m, __double2float_rd(unordered64(s.score[i])));
        s.set[tid] = m;
        if (tid == 0) s.total = 0, s.bound = ~0u;
        __syncthreads();
        const uint64_t least = ordered64((double)bound_of(s, TH, width) - slack);
        for (int i = tid; i < r.n; i += TH) {
            if (s.score[i] < least) continue;
            const int to = atomicAdd(&s.total, 1);
            if (to < ASIDE) s.near_score[to] = s.score[i], s.near_at[to] = s.at[i];
        }
        __syncthreads();
        if (s.total <= ASIDE) r = Ranked{s.near_score, s.near_at, s.total};
    }
    for (int i = tid; i < r.n; i += TH) {
        const uint64_t v = r.score[i], a = r.at[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < r.n; ++j) {
            const uint64_t o = r.score[j];
            rank += o > v || (o == v && r.at[j] < a);
        }
        if (rank < width) s.out_score[rank] = unordered64(v), s.out_at[rank] = a;
    }
    if (tid == 0) s.have = min(r.n, width);
    __syncthreads();
    return r;
}
__device__ __forceinline__ void write_out(const Select& p, int g, const Choice& s, bool bad) {
    for (int w = threadIdx.x; w < p.width; w += TH) {
        const size_t o = (size_t)g * p.width + w;
        const bool some = !bad && w < s.have;
        const int b = some ? (int)(s.out_at[w] >> 32) : -1;
        const int j = some ? (int)(s.out_at[w] & 0x7fffffffu) : 0;
        const bool done = some && over(p, g, b);
        int64_t id = -1;
        if (some)
            id = done ? p.end_id : p.ids ? p.ids[((size_t)g * p.beams + b) * p.ld_ids + j] : j;
        p.out_scores[o] = bad ? NAN : some ? (float)s.out_score[w] : -INFINITY;
        p.out_parents[o] = b;
        p.out_ids[o] = id;
        if (p.out_ended) p.out_ended[o] = some && (done || id == p.end_id);
    }
}

// 2^t within 2^-46 of itself, -1000 <= t < 1000: the Taylor series of e^(f ln 2), |f| <= 1/2, to
// f^11 (what is left out: 0.347^12 / 12! = 6e-15).  Less than half of exp()'s operations,
// on a pipe that such a sum keeps a few multiprocessors busy with.
__device__ __forceinline__ double exp2_series(double t) {
    constexpr double L = sr::LN2;
    constexpr double c2 = L * L / 2, c3 = c2 * L / 3, c4 = c3 * L / 4, c5 = c4 * L / 5, c6 = c5 * L / 6,
                     c7 = c6 * L / 7, c8 = c7 * L / 8, c9 = c8 * L / 9, c10 = c9 * L / 10,
                     c11 = c10 * L / 11;
    t = fmax(t, -1000.0);  // (as good as 0; no branch, so that several run at once)
    const double n = rint(t), f = t - n;
    double y = fma(c11, f, c10);
    y = fma(y, f, c9);
    y = fma(y, f, c8);
    y = fma(y, f, c7);
    y = fma(y, f, c6);
    y = fma(y, f, c5);
    y = fma(y, f, c4);
    y = fma(y, f, c3);
    y = fma(y, f, c2);
    y = fma(y, f, L);
    y = fma(y, f, 1.0);
    return __hiloint2double(__double2hiint(y) + ((int)n << 20), __double2loint(y));
}
// ---- clusters of blocks ----
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address, in the cluster's window, of block `rank`'s copy of `p`.
__device__ __forceinline__ uint32_t address_in(const void* p, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;"
        : "=r"(r)
        : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return r;
}
// A block's share of the sum of 2^((x - top) unit) over chain b's columns, in 64 bits;
// the whole block's, in every thread.  By column, whatever the chain's alignment: equal
// chains have equal sums.
template <typename T>
__device__ __forceinline__ double sum_share(const Select& p, int g, int b, float top, int rank,
                                            int blocks, double* part) {
    const double unit = p.scale * sr::LOG2E;
    const size_t row = (size_t)g * p.beams + b;
    const T* xs = static_cast<const T*>(p.x) + (size_t)g * p.ld_group + (size_t)b * p.ld_beam;
    const int64_t* ids = p.ids ? p.ids + row * p.ld_ids : nullptr;
    const uint32_t* al = p.allowed ? p.allowed + row * p.ld_allowed : nullptr;
    constexpr int AHEAD = 8;  // (loads in flight: one at a time they are what it waits for)
    const int step = blocks * TH;
    double t = 0.0;
    for (long long j0 = rank * TH + (int)threadIdx.x; j0 < p.n; j0 += AHEAD * step) {
        const int j = (int)j0, last = p.n - 1;
        T raw[AHEAD];
        bool in[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            in[a] = j0 + a * step <= last;
            raw[a] = xs[in[a] ? j + a * step : last];
        }
        if (ids) {
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) in[a] &= ids[in[a] ? j + a * step : last] >= 0;
        }
        if (al) {
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int at = in[a] ? j + a * step : last;
                in[a] &= (bool)(al[at >> 5] >> (at & 31) & 1u);
            }
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
            t += in[a] ? exp2_series(((double)to_f32<T>(raw[a]) - (double)top) * unit) : 0.0;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = t;
    __syncthreads();
    t = 0.0;
    for (int i = 0; i < TH / 32; ++i) t += part[i];
    return t;
}
// One block per search, with others of its cluster to help where sums are taken again.
// The chains' normalisers are sums of f32 exponentials, off by up to `slack` / 2: where
// that leaves open which of two chains' columns is the better, among the chosen or at
// their end, the chains' sums are taken again in 64 bits.  Bound by a chain of short
// steps: 6 us for 4 chains of 10000 columns, 8 for 64 x 8 of 131072 (width 64: 13), a
// chain's sum again 14 us by eight blocks, some 50 by one.
struct FinishShared {
    Choice s;
    double sum[MAXW], lse[MAXW], part[TH / 32];
    float top[MAXW];
    unsigned char kind[MAXW], close[MAXW], sure[MAXW];
    double shares[8];  // of the cluster's blocks
    int task;          // the chain whose sum is taken, -1: no more
    float task_top;
};
// The other blocks of a cluster: shares of sums, as long as the first asks for them.
template <typename T>
__device__ __forceinline__ void help_search(const Select& p, FinishShared& f, int g, int rank,
                                            int blocks) {
    const uint32_t task_at = address_in(&f.task, 0), top_at = address_in(&f.task_top, 0);
    const uint32_t share_at = address_in(&f.shares[rank], 0);
    for (;;) {
        cluster_sync();
        int b;
        float top;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(b) : "r"(task_at) : "memory");
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(top) : "r"(top_at) : "memory");
        if (b >= 0) {
            const double t = sum_share<T>(p, g, b, top, rank, blocks, f.part);
            if (threadIdx.x == 0)
                asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(share_at), "d"(t) : "memory");
        }
        cluster_sync();
        if (b < 0) return;
    }
}
template <typename T, bool NORM>
__device__ __forceinline__ void finish_search(const Select& p, const Scan& c, FinishShared& f, int g,
                                              int blocks) {
    Choice& s = f.s;
    double *sum = f.sum, *lse = f.lse;
    float* top = f.top;
    unsigned char *kind = f.kind, *close = f.close, *sure = f.sure;
    const int tid = threadIdx.x, S = c.splits;
    const size_t row0 = (size_t)g * p.beams;
    // ---- the lists, if a thread can hold its share of them: on their way while the
    // chains are looked at (what a chain without columns left is not used) ----
    const int lists = p.beams * S;
    const bool held = lists * p.width <= TH * HELD;
    uint64_t key[HELD];
    int count[HELD];
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const int k = h * TH + tid;
        key[h] = 0, count[h] = 0;
        if (held && k < lists * p.width) {
            key[h] = c.best[row0 * S * p.width + k];
            count[h] = c.part[row0 * S + k / p.width].count;
        }
    }
    // ---- the chains: as many lanes each as they have parts ----
    bool bad = false, again = false;
    int lanes = 1;
    while (lanes < 32 && lanes < S) lanes *= 2;
    for (int b0 = 0; b0 < p.beams; b0 += TH / lanes) {
        const int b = b0 + tid / lanes, lane = tid & (lanes - 1);
        const bool here = b < p.beams;
        const float given = here ? p.beam_scores[row0 + b] : -INFINITY;
        Part mine{0.0, -INFINITY, 0};
        if (here && lane < S) mine = c.part[(row0 + b) * S + lane];
        const int k = here && over(p, g, b) ? OVER : LIVE;
        bad |= !(given < INFINITY);
        double L = 0.0;
        float M = -INFINITY;
        const bool live = k == LIVE && given > -INFINITY;
        int some = 0;  // 1: columns, 2: a sum that is none in f32
        if (live)
            for (int i = lane; i < S; i += lanes) {
                const Part q = i < lanes ? mine : c.part[(row0 + b) * S + i];
                bad |= q.count < 0;
                if (NORM && q.sum > 0.0) M = fmaxf(M, q.m);
                some |= (q.count > 0 ? 1 : 0) | (q.sum == q.sum ? 0 : 2);
            }
        bool lost = false;  // (columns, but a sum of 0 or none)
        if (NORM) {
            for (int o = lanes / 2; o; o >>= 1) {
                M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
                some |= __shfl_xor_sync(0xffffffffu, some, o);
            }
            if (live)
                for (int i = lane; i < S; i += lanes) {
                    const Part q = i < lanes ? mine : c.part[(row0 + b) * S + i];
                    if (q.sum > 0.0)
                        L += q.m == M ? q.sum : q.sum * exp(((double)q.m - (double)M) * p.scale);
                }
            for (int o = lanes / 2; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
            lost = (some & 1) && ((some & 2) || !(L > 0.0));
            if (__any_sync(0xffffffffu, lost)) {
                // (scores out of f32's range: relative to their largest, in 64 bits)
                if (lost) {
                    M = -INFINITY;
                    for (int i = lane; i < S; i += lanes)
                        if (c.part[(row0 + b) * S + i].count > 0)
                            M = fmaxf(M, unordered((uint32_t)(c.best[((row0 + b) * S + i) * p.width] >> 32)));
                    again = true;
                }
                for (int o = lanes / 2; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
            }
        }
        if (lane == 0 && here) {
            sum[b] = given;
            kind[b] = given == -INFINITY ? ABSENT : k;
            lse[b] = L > 0.0 ? (double)M * p.scale + log(L) : 0.0;
            top[b] = M;
            close[b] = NORM && lost;
            sure[b] = 0;
        }
    }
    if (__syncthreads_or(bad)) return write_out(p, g, s, true);

    // candidate `rank` of list i = chain * splits + part; whether there is one
    // (`key` and `count`: as loaded)
    auto worth = [&](int i, int rank, uint64_t key, int count, double& v, int& b, int& j) -> bool {
        b = i / S;
        j = 0;
        v = sum[b];
        if (kind[b] != LIVE) return kind[b] == OVER && rank == 0 && i == b * S;
        if (rank >= count) return false;
        j = (int)~(uint32_t)key;
        v += (double)unordered((uint32_t)(key >> 32)) * p.scale - lse[b];
        return true;
    };
    auto candidate = [&](int i, int rank, double& v, int& b, int& j) -> bool {
        return worth(i, rank, c.best[(row0 * S + i) * p.width + rank], c.part[row0 * S + i].count, v,
                     b, j);
    };
    // the sums of the chains marked, unless they have been taken already; whether one was
    auto sums_again = [&]() -> bool {
        bool more = false;
        for (int b = 0; b < p.beams; ++b) {
            if (!close[b] || sure[b] || kind[b] != LIVE) continue;
            more = true;
            if (!(top[b] > -INFINITY)) continue;  // (no columns)
            if (tid == 0) f.task = b, f.task_top = top[b];
            if (blocks > 1) cluster_sync();
            const double mine = sum_share<T>(p, g, b, top[b], 0, blocks, f.part);
            if (blocks > 1) cluster_sync();
            if (tid == 0) {
                double t = mine;
                for (int i = 1; i < blocks; ++i) t += f.shares[i];
                lse[b] = (double)top[b] * p.scale + log(t);
            }
            __syncthreads();
        }
        for (int b = tid; b < p.beams; b += TH) sure[b] |= close[b];
        __syncthreads();
        return more;
    };
    if (__syncthreads_or(again)) sums_again();
    const double slack = NORM && p.beams > 1 ? (double)c.slack : 0.0;
    for (;;) {
        // What the width-th is not below: of the first q of each list, the width-th (of more
        // than TH lists, of the largest of TH sets).  Few of them, four times the width, if
        // that saves sorting them (see bound_of), else TH: one chain may hold all the best
        // (12 x 32 x 14365, width 32: with twice the width 38 us, 24 so).
        const int few = p.width <= 8 ? (4 * p.width + lists - 1) / lists : TH;
        const int q = max(1, min(few, min(TH / lists, p.width)));
        if (tid == 0) s.count = 0, s.bound = ~0u;
        bool dropped = false;
        if (held) {
            double v[HELD];
            int b[HELD], col[HELD];
#pragma unroll
            for (int h = 0; h < HELD; ++h) {
                const int k = h * TH + tid, i = k / p.width, rank = k - i * p.width;
                if (i >= lists || !worth(i, rank, key[h], count[h], v[h], b[h], col[h]))
                    v[h] = -INFINITY;
                if (lists <= TH && i < lists && rank < q) s.set[i * q + rank] = __double2float_rd(v[h]);
            }
            if (lists > TH) {
                float m = -INFINITY;
#pragma unroll
                for (int h = 0; h < HELD; ++h) m = fmaxf(m, __double2float_rd(v[h]));
                s.set[tid] = m;
            }
            pick(s, v, b, col, min(lists * q, TH), p.width, slack);
        } else {
            float m = -INFINITY;
            for (int k = tid; k < lists * q; k += TH) {
                double v;
                int b, j;
                if (candidate(k / q, k % q, v, b, j)) m = fmaxf(m, __double2float_rd(v));
            }
            s.set[tid] = m;
            __syncthreads();
            double least = (double)bound_of(s, min(lists * q, TH), p.width) - slack;
            // ---- the lists, so many ranks at a time, until none reaches it ----
            const int some = min(lists, ROUND), ranks = max(1, ROUND / some);
            for (int r0 = 0; r0 < p.width; r0 += ranks) {
                bool any = false;
                for (int l0 = 0; l0 < lists; l0 += some) {
#pragma unroll 4
                    for (int k = tid; k < some * ranks; k += TH) {
                        const int i = l0 + k / ranks, rank = r0 + k % ranks;
                        double v;
                        int b, j;
                        if (i < lists && rank < p.width && candidate(i, rank, v, b, j) && v >= least)
                            add(s, v, b, j), any = true;
                    }
                    __syncthreads();
                    if (s.count > CAP - ROUND) {  // (what is just behind the width-th is dropped)
                        rank_all(s, p.width, 0.0);
                        for (int w = tid; w < s.have; w += TH)
                            s.score[w] = ordered64(s.out_score[w]), s.at[w] = s.out_at[w];
                        if (tid == 0) s.count = s.have;
                        if (s.have == p.width) least = s.out_score[p.width - 1] - slack;
                        dropped = true;
                    }
                    __syncthreads();
                }
                if (!__syncthreads_or(any)) break;
            }
        }
        const Ranked r = rank_all(s, p.width, slack);
        if (slack == 0.0) break;
        // ---- is their order sure? ----
        const int have = s.have;
        for (int w = tid; w + 1 < have; w += TH) {
            const int a = (int)(s.out_at[w] >> 32), b = (int)(s.out_at[w + 1] >> 32);
            if (a != b && s.out_score[w] - s.out_score[w + 1] <= slack) close[a] = close[b] = 1;
        }
        if (have == p.width) {
            const double last = s.out_score[have - 1];
            const uint64_t last_at = s.out_at[have - 1];
            const int a = (int)(last_at >> 32);
            for (int i = tid; i < r.n; i += TH) {
                const double v = unordered64(r.score[i]);
                const int b = (int)(r.at[i] >> 32);
                const bool behind = v < last || (v == last && r.at[i] > last_at);
                if (behind && b != a && last - v <= slack) close[a] = close[b] = 1;
            }
        }
        if (dropped)
            for (int b = tid; b < p.beams; b += TH) close[b] = 1;
        __syncthreads();
        if (!sums_again()) break;
    }
    write_out(p, g, s, false);
}

template <typename T, bool NORM, bool GATE>
__global__ void __launch_bounds__(TH, 4) scan_kernel(const Select p, const Scan c) {
    extern __shared__ uint4 scan_raw[];
    const size_t row = blockIdx.x / c.splits;
    const int g = (int)(row / p.beams), b = (int)(row % p.beams);
    if (over(p, g, b) || absent(p, g, b)) return;
    scan_part<T, NORM, GATE>(p, c, *reinterpret_cast<ScanShared<T>*>(scan_raw), row,
                             blockIdx.x % c.splits, g, b);
}
template <typename T, bool NORM>
__global__ void __launch_bounds__(TH, 4) finish_kernel(const Select p, const Scan c, int blocks) {
    __shared__ FinishShared f;
    const int g = blockIdx.x / blocks, rank = blockIdx.x % blocks;  // (a cluster's blocks lie side by side)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (rank > 0) return help_search<T>(p, f, g, rank, blocks);
    finish_search<T, NORM>(p, c, f, g, blocks);
    if (blocks > 1) {
        __syncthreads();
        if (threadIdx.x == 0) f.task = -1;
        cluster_sync();
        cluster_sync();  // (the others have read it)
    }
}

// One block per search whose columns are CAP at most in all: their normalisers in 64
// bits, a warp per chain, and the best, a thread's share of the columns in registers.
template <typename T>
__global__ void __launch_bounds__(TH, 4) small_kernel(const Select p) {
    constexpr int H = CAP / TH;
    __shared__ Choice s;
    __shared__ double lse[MAXW];
    const int tid = threadIdx.x, lane = tid & 31, g = blockIdx.x;
    const size_t row0 = (size_t)g * p.beams;
    if (tid == 0) s.count = 0, s.bound = ~0u;
    if (p.normalise) {
        for (int b = tid >> 5; b < p.beams; b += TH / 32) {
            if (absent(p, g, b) || over(p, g, b)) continue;
            double m = -INFINITY, t = 0.0;
            for (int j = lane; j < p.n; j += 32) m = fmax(m, p.scale * column<T>(p, g, b, j));
#pragma unroll
            for (int o = 16; o; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (m > -INFINITY)
                for (int j = lane; j < p.n; j += 32) t += exp(p.scale * column<T>(p, g, b, j) - m);
#pragma unroll
            for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
            if (lane == 0) lse[b] = m > -INFINITY ? m + log(t) : 0.0;
        }
        __syncthreads();
    }
    bool bad = false;
    double v[H];
    int b[H], j[H];
    const int all = p.beams * p.n;
#pragma unroll
    for (int h = 0; h < H; ++h) {
        const int k = h * TH + tid;
        v[h] = -INFINITY;
        if (k >= all) continue;
        b[h] = k / p.n, j[h] = k - b[h] * p.n;
        const float given = p.beam_scores[row0 + b[h]];
        const double x = p.scale * column<T>(p, g, b[h], j[h]);
        bad |= !(given < INFINITY);
        if (given == -INFINITY) continue;
        if (over(p, g, b[h])) {
            if (j[h] == 0) v[h] = given;
        } else {
            bad |= !(x < INFINITY);
            if (x > -INFINITY) v[h] = (double)given + (p.normalise ? x - lse[b[h]] : x);
        }
    }
    bad = __syncthreads_or(bad);
    if (!bad) {
        float m = -INFINITY;
#pragma unroll
        for (int h = 0; h < H; ++h) m = fmaxf(m, __double2float_rd(v[h]));
        s.set[tid] = m;
        pick(s, v, b, j, min(all, TH), p.width, 0.0);
        rank_all(s, p.width, 0.0);
    }
    write_out(p, g, s, bad);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
struct Plan {
    bool small;
    Scan c;
    size_t bytes;
};
static Plan plan(const Ctx& c, const fdb_beam_args& a) {
    Plan p{};
    p.small = a.beams * a.n <= CAP;
    if (p.small) return p;
    const size_t rows = a.groups * a.beams, per = a.dtype == FDB_DTYPE_F32 ? 4 : 8;
    // Blocks that are all resident at once (four a multiprocessor), of a tile or more: a
    // block starts and ends with some 4 us in which it loads nothing (512 chains of 131072
    // bf16: 29.9 us with a block each, 31.8 with two, 36 with three).
    const size_t vecs = a.n / per + 2;  // (at most)
    const size_t most = (vecs + TH * U - 1) / (TH * U);
    const size_t least = (most + SPANS * SPAN - 1) / (SPANS * SPAN);
    // And no more lists than a block of the finish holds in registers, even where that leaves
    // multiprocessors idle: of 1 to 4 searches of 4 to 64 chains of 131072 columns, widths 8 to
    // 64, all but a few are slower with more parts, read by the finish's second form (1 x 32,
    // width 32, f32: 26.5 us, 30.7 with parts for all; 1 x 8, width 8: 16.2, 21.6, and 20.1 with
    // a block a multiprocessor), and those few within 2 us.
    const size_t lists = std::max<size_t>(1, TH * HELD / (a.beams * a.width));
    p.c.splits = (int)std::max(least, std::min({most, lists, std::max<size_t>(1, (size_t)c.sm_count * 4 / rows)}));
    Carve ws(a.workspace);
    p.c.part = ws.take<Part>(rows * p.c.splits);
    p.c.best = ws.take<uint64_t>(rows * p.c.splits * a.width);
    p.bytes = ws.at;
    return p;
}
size_t select_bytes(const Ctx& c, const fdb_beam_args& a) { return plan(c, a).bytes; }

template <typename T, bool NORM, bool GATE>
static void launch_scan(cudaStream_t s, int device, unsigned blocks, const Select& p, const Scan& c) {
    constexpr size_t smem = sizeof(ScanShared<T>);
    static std::atomic<uint64_t> done{0};
    sr::allow_smem(scan_kernel<T, NORM, GATE>, device, smem, done);
    scan_kernel<T, NORM, GATE><<<blocks, TH, smem, s>>>(p, c);
    FDB_LAUNCH_CHECK();
}
template <typename T, bool NORM>
static void run(const Ctx& ctx, const fdb_beam_args& a, const Select& p, const Scan& c) {
    const cudaStream_t s = static_cast<cudaStream_t>(a.stream);
    FDB_REQUIRE(a.groups * a.beams * c.splits < (1ull << 31), FDB_ERR_INVALID_ARG, "too many chains");
    const unsigned parts = (unsigned)(a.groups * a.beams * c.splits);
    if (a.ids || a.allowed) launch_scan<T, NORM, true>(s, ctx.device, parts, p, c);
    else launch_scan<T, NORM, false>(s, ctx.device, parts, p, c);
    // Launched while the scan ends; blocks that help, where there is room for them.
    unsigned blocks = 1;
    while (NORM && a.beams > 1 && blocks < 8 && a.groups * blocks * 2 <= (size_t)ctx.sm_count * 4) blocks *= 2;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = blocks, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t how{};
    how.gridDim = dim3((unsigned)a.groups * blocks), how.blockDim = dim3(TH), how.stream = s;
    how.attrs = attr, how.numAttrs = 2;
    FDB_CUDA(cudaLaunchKernelEx(&how, finish_kernel<T, NORM>, p, c, (int)blocks));
}
template <typename T>
static void run(const Ctx& ctx, const fdb_beam_args& a, const Select& p) {
    Plan l = plan(ctx, a);
    if (l.small) {
        small_kernel<T><<<(unsigned)a.groups, TH, 0, static_cast<cudaStream_t>(a.stream)>>>(p);
        FDB_LAUNCH_CHECK();
        return;
    }
    l.c.s = (float)std::min((double)a.scale * sr::LOG2E, 3e38);
    // What two normalisers may be off by.  Each term: its exponential and up to three
    // factors that are exponentials (2^-22 each), ten additions (2^-24), and in the
    // exponent the product's rounding and that of s (2 x 2^-24 of it, times ln 2); the
    // sum sees the exponents' mean under the softmax, at most their entropy, log2 n, and
    // the 8 that a reference may lie below the largest.
    l.c.slack = (float)(2.0 * (0x1p-20 + 10 * 0x1p-24 +
                               1.4 * 0x1p-24 * (std::log2((double)a.n) + 8.0)));
    if (a.normalise) run<T, true>(ctx, a, p, l.c);
    else run<T, false>(ctx, a, p, l.c);
}
void select_run(const Ctx& ctx, const fdb_beam_args& a) {
    Select p{};
    p.x = a.scores;
    p.beams = (int)a.beams, p.n = (int)a.n, p.width = (int)a.width;
    p.ld_group = a.ld_group, p.ld_beam = a.ld_beam;
    p.scale = a.scale, p.normalise = a.normalise != 0;
    p.ids = a.ids, p.ld_ids = a.ld_ids;
    p.allowed = a.allowed, p.ld_allowed = a.allowed ? a.ld_allowed : 0;
    p.beam_scores = a.beam_scores, p.ended = a.ended, p.end_id = a.end_id;
    p.out_scores = a.out_scores, p.out_parents = a.out_parents, p.out_ids = a.out_ids;
    p.out_ended = a.out_ended;
    if (a.dtype == FDB_DTYPE_F32) run<float>(ctx, a, p);
    else if (a.dtype == FDB_DTYPE_F16) run<__half>(ctx, a, p);
    else run<__nv_bfloat16>(ctx, a, p);
}

// ---------------------------------------------------------------------------
// states
// ---------------------------------------------------------------------------
// All states of a call in one launch (STATES of them).  Out of place a warp moves 4 KB
// of a run, eight loads a lane in flight, or, of runs that are shorter, several.  In
// place a thread takes 16 bytes of every row of a search, all of them before it writes
// any; rows that stay where they are are not touched.  Out of place bound by memory (6.6
// TB/s).  In place by the loads in flight, fewer as a thread holds more rows: 512 rows of 512
// KB in all moved at 5.5 TB/s by searches of 8 beams, 4.1 of 16, 2.5 of 32, 0.8 of 128.
constexpr int STATES = 64;
constexpr int PIECE = 8;                 // vectors of a lane
struct State {
    const unsigned char* src;
    unsigned char* dst;
    size_t src_stride, dst_stride, src_part, dst_part;
    size_t vecs;                         // of a run
    unsigned parts, runs, pieces, first; // first: unit of the launch
    int vec, lanes;                      // log2 of a vector's bytes, of a run's lanes
};
struct States {
    State e[STATES];
    int count;
};
__device__ __forceinline__ const State& state_of(const States& t, unsigned unit) {
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.e[mid].first <= unit) lo = mid;
        else hi = mid;
    }
    return t.e[lo];
}
template <typename V>
__device__ __forceinline__ void move_run(const State& t, unsigned unit, int lane,
                                         const int64_t* __restrict__ parents, unsigned beams,
                                         unsigned width, int clear) {
    const unsigned piece = unit % t.pieces;
    const unsigned run = (unit / t.pieces << (5 - t.lanes)) + (lane >> t.lanes);
    if (run >= t.runs) return;
    const unsigned row = run / t.parts, part = run % t.parts;
    const int64_t from = parents[row];
    const bool none = (uint64_t)from >= beams;
    if (none && !clear) return;
    const size_t at = (size_t)(row / width) * beams + (none ? 0 : (size_t)from);
    const V* s = reinterpret_cast<const V*>(t.src + at * t.src_stride + part * t.src_part);
    V* d = reinterpret_cast<V*>(t.dst + row * t.dst_stride + part * t.dst_part);
    const size_t v0 = (size_t)piece * (32 * PIECE) + (lane & ((1 << t.lanes) - 1));
    s += v0, d += v0;
    const int left = (int)min(t.vecs - min(v0, t.vecs), (size_t)32 * PIECE);
    V r[PIECE];
    if (left > 32 * (PIECE - 1) && !none) {
#pragma unroll
        for (int k = 0; k < PIECE; ++k) r[k] = __ldcs(s + 32 * k);
#pragma unroll
        for (int k = 0; k < PIECE; ++k) __stcs(d + 32 * k, r[k]);
        return;
    }
#pragma unroll
    for (int k = 0; k < PIECE; ++k) {
        r[k] = V();
        if (32 * k < left && !none) r[k] = __ldcs(s + 32 * k);
    }
#pragma unroll
    for (int k = 0; k < PIECE; ++k)
        if (32 * k < left) d[32 * k] = r[k];
}
__global__ void __launch_bounds__(256)
    move_kernel(const __grid_constant__ States t, const int64_t* __restrict__ parents,
                unsigned beams, unsigned width, int clear, unsigned units) {
    const unsigned u = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (u >= units) return;
    const State& e = state_of(t, u);
    const unsigned unit = u - e.first;
    if (e.vec == 4) move_run<uint4>(e, unit, lane, parents, beams, width, clear);
    else if (e.vec == 3) move_run<uint2>(e, unit, lane, parents, beams, width, clear);
    else if (e.vec == 2) move_run<unsigned>(e, unit, lane, parents, beams, width, clear);
    else if (e.vec == 1) move_run<unsigned short>(e, unit, lane, parents, beams, width, clear);
    else move_run<unsigned char>(e, unit, lane, parents, beams, width, clear);
}
template <typename V>
__device__ __forceinline__ void turn_run(const State& t, unsigned unit, const int* from, int beams,
                                         unsigned char* held_raw) {
    V* held = reinterpret_cast<V*>(held_raw) + threadIdx.x;  // [beams][threads]
    const unsigned piece = unit % t.pieces, run = unit / t.pieces;
    const size_t g = run / t.parts, part = run % t.parts;
    const size_t v = (size_t)piece * blockDim.x + threadIdx.x;
    if (v >= t.vecs) return;
    unsigned char* c = t.dst + g * beams * t.dst_stride + part * t.dst_part + v * sizeof(V);
#pragma unroll 4
    for (int b = 0; b < beams; ++b)
        if (from[b] >= 0)
            held[b * blockDim.x] = *reinterpret_cast<const V*>(c + (size_t)from[b] * t.dst_stride);
#pragma unroll 4
    for (int b = 0; b < beams; ++b)
        if (from[b] >= 0) *reinterpret_cast<V*>(c + (size_t)b * t.dst_stride) = held[b * blockDim.x];
}
__global__ void turn_kernel(const __grid_constant__ States t, const int64_t* __restrict__ parents,
                            int beams) {
    extern __shared__ uint4 held[];
    __shared__ int from[MAXW];  // the row that comes, -1: it stays as it is
    const State& e = state_of(t, blockIdx.x);
    const unsigned unit = blockIdx.x - e.first;
    const size_t g = unit / e.pieces / e.parts;
    for (int b = threadIdx.x; b < beams; b += blockDim.x) {
        const int64_t f = parents[g * beams + b];
        from[b] = (uint64_t)f < (uint64_t)beams && f != b ? (int)f : -1;
    }
    __syncthreads();
    unsigned char* h = reinterpret_cast<unsigned char*>(held);
    if (e.vec == 4) turn_run<uint4>(e, unit, from, beams, h);
    else if (e.vec == 3) turn_run<uint2>(e, unit, from, beams, h);
    else if (e.vec == 2) turn_run<unsigned>(e, unit, from, beams, h);
    else if (e.vec == 1) turn_run<unsigned short>(e, unit, from, beams, h);
    else turn_run<unsigned char>(e, unit, from, beams, h);
}

void reorder_run(const Ctx& c, const fdb_beam_state* states, size_t count,
                 const fdb_reorder_opts& o) {
    const cudaStream_t s = static_cast<cudaStream_t>(o.stream);
    // threads that fit into 48 KB with 16 bytes of every row each
    const int turn_threads = (int)std::max<size_t>(32, std::min<size_t>(256, 49152 / (16 * o.beams) / 32 * 32));
    States move{}, turn{};
    unsigned long long move_units = 0, turn_units = 0;
    auto flush_move = [&] {
        if (move.count)
            move_kernel<<<(unsigned)((move_units + 7) / 8), 256, 0, s>>>(
                move, o.parents, (unsigned)o.beams, (unsigned)o.width, o.clear, (unsigned)move_units);
        FDB_LAUNCH_CHECK();
        move.count = 0, move_units = 0;
    };
    auto flush_turn = [&] {
        if (turn.count) {
            const size_t smem = (size_t)turn_threads * o.beams * 16;
            if (smem > 40960) {  // (with the static part, over what needs no permission)
                static std::atomic<uint64_t> done{0};
                sr::allow_smem(turn_kernel, c.device, 65536, done);
            }
            turn_kernel<<<(unsigned)turn_units, turn_threads, smem, s>>>(turn, o.parents,
                                                                         (int)o.beams);
        }
        FDB_LAUNCH_CHECK();
        turn.count = 0, turn_units = 0;
    };
    // (all of them looked at before the first is moved)
    std::vector<State> all;
    all.reserve(count);
    for (size_t i = 0; i < count; ++i) {
        const fdb_beam_state& a = states[i];
        if (a.bytes == 0 || a.parts == 0) continue;
        const bool here = a.src == a.dst;
        State t{};
        t.src = static_cast<const unsigned char*>(a.src), t.dst = static_cast<unsigned char*>(a.dst);
        t.src_stride = a.src_stride, t.dst_stride = a.dst_stride;
        t.src_part = a.src_part_stride, t.dst_part = a.dst_part_stride;
        size_t bytes = a.bytes, parts = a.parts;
        if (parts > 1 && t.dst_part == bytes && (here || t.src_part == bytes))
            bytes *= parts, parts = 1;  // (runs without gaps are one)
        uintptr_t bits = reinterpret_cast<uintptr_t>(a.src) | reinterpret_cast<uintptr_t>(a.dst) |
                         t.src_stride | t.dst_stride | bytes;
        if (parts > 1) bits |= t.src_part | t.dst_part;
        while (t.vec < 4 && !(bits >> t.vec & 1)) ++t.vec;
        t.vecs = bytes >> t.vec;
        t.parts = (unsigned)parts;
        const size_t runs = (here ? o.groups : o.groups * o.width) * parts;
        t.lanes = 5;
        while (!here && t.lanes > 0 && t.vecs <= (size_t)1 << (t.lanes - 1)) --t.lanes;
        const size_t piece = here ? (size_t)turn_threads : t.lanes < 5 ? t.vecs : 32 * PIECE;
        const size_t pieces = (t.vecs + piece - 1) / piece;
        const unsigned long long groups = here ? runs : (runs + (32u >> t.lanes) - 1) >> (5 - t.lanes);
        FDB_REQUIRE(runs < (1ull << 31) && pieces < (1ull << 31) && groups * pieces < (1ull << 31),
                    FDB_ERR_INVALID_ARG, "a state is too large");
        t.runs = (unsigned)runs, t.pieces = (unsigned)pieces;
        t.first = (unsigned)(groups * pieces);  // (its units, until it has a place)
        all.push_back(t);
    }
    for (State& t : all) {
        const bool here = t.src == t.dst;
        States& table = here ? turn : move;
        unsigned long long& units = here ? turn_units : move_units;
        if (table.count == STATES || units + t.first >= (1ull << 31)) {
            if (here) flush_turn();
            else flush_move();
        }
        const unsigned mine = t.first;
        t.first = (unsigned)units;
        table.e[table.count++] = t;
        units += mine;
    }
    flush_move();
    flush_turn();
}

}  // namespace beam
}  // namespace fdb
