// softmax_rows.cu -- log probabilities under a softmax over index rows, and
// their gradient, without ever holding the nq x n scores.
//
//   s_ij = scale * q_i . x_j         over the rows j that query i may see
//   lse_i = log sum_j exp(s_ij),  p_ij = exp(s_ij - lse_i)
//   H_i = lse_i - sum_j p_ij s_ij,  logprob_i = s_i,t(i) - lse_i
//
// Forward: the scores are formed tile by tile on the tensor cores (or, for a
// few queries, on the FMA pipes) and every thread folds its columns into
// a running (max m, sum l = sum 2^(t - m), a = sum 2^(t - m) (t - m)) of its
// query row, t = s log2(e); the partial triples are joined by
// finish_kernel:  lse = ln2 (M + log2 L),  H = ln2 (log2 L - A / L).
// For the top alternatives each group of 32 rows leaves its largest score,
// the pair of rows that holds it (in the low 4 bits) and its second largest;
// a little more than the best k groups are picked per query, their marked rows
// are scored again exactly (64-bit sums), and a group whose second largest
// could still enter is scored in full, as are all groups if one that was not
// picked could.
// Which ids are returned therefore does not depend on the order of a 32-bit
// sum (but see may_enter); equal scores go to the lower id.
//
// Types: 16-bit rows go to the MMA as they are.  f32 rows are split once into
// two fp16 parts of the row scaled by a power of two, x 2^e = hi + lo
// (22 bits, the row's largest element at 2^14), and a score is the sum of
// three products lo.hi + hi.lo + hi.hi, the small ones first: the tensor
// core's accumulation cuts bits off the running sum, so its size should be
// small for as long as possible.  lo.lo (2^-22 of the score) is left out.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "fdb_internal.h"
#include "softmax_rows.cuh"
#include "tc_ptx.cuh"

namespace fdb {
namespace sr {

using namespace tc;

constexpr int BM = 128;                     // rows of an output tile in one block
constexpr int PM = 2 * BM;                  // ... of the pair of blocks that shares it
constexpr int OPER = BM * 128;              // bytes of 128 rows of a 64-wide K step
// Two blocks work on a tile as a pair (cta_group::2): each holds its 128 rows
// of A and half of the columns' rows of B, so an operand byte is fetched and
// read from shared memory half as often for B.  Whole sums: 256 columns an
// accumulator, six K steps of 32 KB a block in flight.  Sums in blocks (see
// rows_kernel): 128 columns; two parts (f32) have four K steps of 48 KB (both
// parts of both operands), one part eight of 24 KB.  GRAD has one stage less
// of either: its output is staged in shared memory too.  Two parts of at most
// 128 of K are one block anyway: whole sums of 256 columns, three K steps of
// 64 KB.
__host__ __device__ constexpr int bn_of(bool blk) { return blk ? 128 : 256; }
__host__ __device__ constexpr int stages_of(bool two, bool blk, bool grad) {
    return two && !blk ? 3 : (two ? 4 : blk ? 8 : 6) - (grad ? 1 : 0);
}
__host__ __device__ constexpr int stage_bytes(bool two, bool blk) {
    return (two ? 2 : 1) * (OPER + bn_of(blk) / 2 * 128);
}
__host__ __device__ constexpr int accs_of(bool blk) { return blk ? 4 : 2; }
constexpr int STAGED = 32 * 64;             // one warp's 32 x 32 fp16 outputs
__host__ __device__ constexpr int staged_of(bool two, bool grad) {
    return grad ? 16 * (two ? 2 : 1) * STAGED : 0;
}
constexpr int MAX_STG = 8;
// K steps of an accumulator, sums in blocks
__host__ __device__ constexpr int kblock_of(bool two, bool grad) { return !two ? 4 : grad ? 1 : 2; }
constexpr int MAX_BN = 256;
constexpr unsigned long long DRAIN_CYCLES = 4000000ull;  // about 2 ms
constexpr int THREADS = 640;                // 2 issuing warps, 2 idle, 16 epilogue warps
constexpr int EPI_WARP0 = 4, EPI_WARPS = 16;
constexpr int GROUP = 32;                   // rows whose largest scores are kept together
// Groups picked beyond k: what the bound then lies below the kth score by has to
// exceed the errors of 32-bit scores, else all groups are looked at.  Of random
// scores 4 places are some hundred times that (8: 2048 x 131072 x 768, k = 20
// takes 108 us instead of 99).
constexpr int PAD = 4;
static_assert(FDB_MAX_ALTERNATIVES + PAD <= 128, "the bound is one of 128 maxima");
constexpr float NONE = -1e30f;              // score of a row that may not be seen
constexpr float NONE_BELOW = -1e29f;
constexpr float RAISE = 8.0f;               // see Run

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// A running (reference m, sum l = sum 2^(t - m), a = sum 2^(t - m) (t - m)) of
// one query's columns, t = score * log2(e), in f32: the sums of 32 columns each are
// added one after the other, a quarter of a unit's column tiles to a thread (at
// most some 10^4 of them for a million rows: their roundings, of either sign, come
// to a few 1e-6 of the sum).  m starts at the first columns'
// largest t and is raised only when a t exceeds it by more than RAISE: the
// sums then hold terms of at most 2^8 (f32's relative precision does not
// care), and a new largest score seldom costs a rescaling.
struct Run {
    float m, l, a;
    float limit;  // -inf before the first columns, then RAISE
};
__device__ __forceinline__ Run run_empty() { return Run{0.0f, 0.0f, 0.0f, -INFINITY}; }
// For columns with largest t - m = cm: what t - m loses (0 mostly).
__device__ __forceinline__ float run_raise(Run& r, float cm) {
    if (!(cm > r.limit && cm > NONE_BELOW)) return 0.0f;
    const float m = r.m + cm, d = m - r.m;  // (d: what m moved by after rounding)
    r.m = m;
    r.limit = RAISE;
    if (!(r.l == 0.0f && r.a == 0.0f)) {
        const float f = ex2(-d);
        r.a = __fmaf_rn(-d, r.l, r.a) * f;
        r.l *= f;
    }
    return d;
}
__device__ __forceinline__ void run_join(Run& r, Run o) {
    if (o.limit == -INFINITY) return;
    if (r.limit == -INFINITY || o.m > r.m) {
        const Run t = r;
        r = o;
        o = t;
    }
    if (!(o.l == 0.0f && o.a == 0.0f)) {
        const float d = o.m - r.m, f = ex2(d);
        r.a += __fmaf_rn(d, o.l, o.a) * f;
        r.l += o.l * f;
    }
}
// As stored: m is -inf for a run without columns; top is the largest score of
// its groups.
__device__ __forceinline__ float4 run_stored(const Run& r, float top) {
    return make_float4(r.limit == -INFINITY ? -INFINITY : r.m, r.l, r.a, top);
}

// A group's largest score without the mark of its pair.
__device__ __forceinline__ float unmarked(float f) {
    return __uint_as_float(__float_as_uint(f) & ~15u);
}
// The largest of 32 values with the number of its pair in the low 4 bits, and
// the second largest (either may be moved by the marks: 2^-19 relative).
__device__ __forceinline__ float2 top_pair(const float (&u)[32]) {
    // four running (largest, second) pairs: an operation for the second, as
    // there is a maximum of three
    float m1[4], m2[4];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int c = i & 3;
        const float hi = __uint_as_float(
            (__float_as_uint(fmaxf(u[2 * i], u[2 * i + 1])) & ~15u) | (unsigned)i);
        const float lo = fminf(u[2 * i], u[2 * i + 1]);
        if (i < 4) {
            m1[c] = hi;
            m2[c] = lo;
        } else {
            m2[c] = max3(m2[c], lo, fminf(m1[c], hi));
            m1[c] = fmaxf(m1[c], hi);
        }
    }
#pragma unroll
    for (int w = 2; w >= 1; w >>= 1)
#pragma unroll
        for (int c = 0; c < w; ++c) {
            m2[c] = max3(m2[c], m2[c + w], fminf(m1[c], m1[c + w]));
            m1[c] = fmaxf(m1[c], m1[c + w]);
        }
    return make_float2(m1[0], m2[0]);
}

// ---------------------------------------------------------------------------
// packing
// ---------------------------------------------------------------------------
// One warp per row: f32 (or 16-bit) values scaled by 2^e, |largest| in
// [2^13, 2^14), as fp16 hi and, with two parts, lo = the rest; columns padded
// with zeros to kp.  f[row] = 2^-e; 0 for a row of zeros, NaN for a row with
// an infinity or NaN (its elements are then written as zeros: the NaN reaches
// a score through f alone, so a query that may not see the row is not
// touched).  `seen` (nullable): rows whose bit is clear are taken as zeros.
// Bound by memory: reads d * size, writes 2 * parts * kp a row; rows of up to
// 4 vectors (or, unaligned, 14 pairs) a lane stay in registers between the two
// passes.
struct PackSide {
    const void* x;
    size_t ld;
    int n;
    const uint32_t* seen;
    const float* lse;    // nullable: a row whose lse is -inf counts as zeros, too
    __half* out;
    float* f;
    unsigned* largest;   // see most_of, nullable
    const int* weight;   // nullable
    int blocks;          // of 8 warps
    int rows;            // a warp's: 4 short ones (512 bytes at most) or 1
    int wide;            // rows can be read in 16-byte vectors
};
// What the largest is taken of: the scales' bits, or, with weights, WEIGHT_ZERO + the
// exponent of scale times weight; 0 is none.
constexpr int WEIGHT_ZERO = 1024;
__device__ __forceinline__ unsigned most_of(const PackSide& p, int row, float f) {
    if (!p.largest || !(f > 0.0f)) return 0u;
    if (!p.weight) return __float_as_uint(f);
    const int w = p.weight[row];
    return w == NO_WEIGHT ? 0u : (unsigned)(ilogbf(f) + w + WEIGHT_ZERO);
}
template <typename T, int PARTS>
__device__ __forceinline__ unsigned pack_row(const PackSide& p, int row, int d, int kp) {
    constexpr int V = 16 / (int)sizeof(T), NV = 4, NP = 14;
    const int lane = threadIdx.x & 31;
    const T* src = static_cast<const T*>(p.x) + (size_t)row * p.ld;
    __half* dst = p.out + (size_t)row * (size_t)(PARTS * kp);
    const bool use = (!p.seen || (p.seen[row >> 5] >> (row & 31) & 1u)) &&
                     (!p.lse || p.lse[row] != -INFINITY);
    const bool held = p.wide && d <= 32 * V * NV;
    const bool pairs = !held && d <= 64 * NP;  // two columns a lane and step
    uint4 raw[NV];
    float two[2 * NP];
    float mx = 0.0f;
    bool bad = false;
    if (use && held) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * 32 + lane) * V;
            raw[i] = make_uint4(0, 0, 0, 0);
            if (c < d) raw[i] = __ldg(reinterpret_cast<const uint4*>(src + c));
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const T* e = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float v = fabsf(to_f32<T>(e[j]));
                bad |= !(v <= FLT_MAX);
                mx = fmaxf(mx, v);
            }
        }
    } else if (use && pairs) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int c = i * 64 + 2 * lane;
            two[2 * i] = c < d ? to_f32<T>(src[c]) : 0.0f;
            two[2 * i + 1] = c + 1 < d ? to_f32<T>(src[c + 1]) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 2 * NP; ++i) {
            const float v = fabsf(two[i]);
            bad |= !(v <= FLT_MAX);
            mx = fmaxf(mx, v);
        }
    } else if (use) {
        for (int c = lane; c < d; c += 32) {
            const float v = fabsf(to_f32<T>(src[c]));
            bad |= !(v <= FLT_MAX);
            mx = fmaxf(mx, v);
        }
    }
    bad = __any_sync(0xffffffffu, bad);
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    // 2^e with mx 2^e in [2^13, 2^14); e within +-120 keeps 2^e and 2^-e normal
    int e = 0;
    if (!bad && mx > 0.0f) e = max(-120, min(120, 13 - ilogbf(mx)));
    const float s = ldexpf(1.0f, e);
    const bool zero = bad || !(mx > 0.0f);
    if (held) {  // (d is a multiple of V, kp of 16: whole vectors, zeros past d)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * 32 + lane) * V;
            if (c >= kp) break;
            const T* x = reinterpret_cast<const T*>(&raw[i]);
            __align__(16) __half hi[V], lo[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float v = !zero && c < d ? to_f32<T>(x[j]) * s : 0.0f;
                hi[j] = __float2half_rn(v);
                lo[j] = __float2half_rn(v - __half2float(hi[j]));
            }
            if (V == 8) {
                *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(hi);
            } else {
                *reinterpret_cast<uint2*>(dst + c) = *reinterpret_cast<const uint2*>(hi);
                if (PARTS == 2)
                    *reinterpret_cast<uint2*>(dst + kp + c) = *reinterpret_cast<const uint2*>(lo);
            }
        }
    } else if (pairs) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int c = i * 64 + 2 * lane;
            if (c >= kp) break;
            const float a = zero ? 0.0f : two[2 * i] * s, b = zero ? 0.0f : two[2 * i + 1] * s;
            const __half2 hi = __floats2half2_rn(a, b);
            *reinterpret_cast<__half2*>(dst + c) = hi;
            if (PARTS == 2) {
                const float2 back = __half22float2(hi);
                *reinterpret_cast<__half2*>(dst + kp + c) =
                    __floats2half2_rn(a - back.x, b - back.y);
            }
        }
    } else {
        for (int c = lane; c < kp; c += 32) {
            const float v = (!zero && c < d) ? to_f32<T>(src[c]) * s : 0.0f;
            const __half hi = __float2half_rn(v);
            dst[c] = hi;
            if (PARTS == 2) dst[kp + c] = __float2half_rn(v - __half2float(hi));
        }
    }
    const float r = bad ? __int_as_float(0x7fc00000) : (mx > 0.0f ? ldexpf(1.0f, -e) : 0.0f);
    if (lane == 0) p.f[row] = r;
    return most_of(p, row, r);
}
// Rows of one vector a lane at most, four at a time: a warp that waits for one
// such row after the other has too little in flight (262144 x 96 f32: 85 us,
// four at a time 43).  Rows that are not aligned are read an element at a time
// (198627 x 25 f32: 81 us one row at a time, 37 so).
template <typename T, int PARTS, bool WIDE>
__device__ __forceinline__ unsigned pack_short(const PackSide& p, int row0, int d, int kp) {
    constexpr int V = 16 / (int)sizeof(T), R = 4;
    const int lane = threadIdx.x & 31, c = lane * V;
    uint4 raw[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = row0 + r;
        raw[r] = make_uint4(0, 0, 0, 0);
        const bool use = row < p.n && (!p.seen || (p.seen[row >> 5] >> (row & 31) & 1u)) &&
                         (!p.lse || p.lse[row] != -INFINITY);
        const T* src = static_cast<const T*>(p.x) + (size_t)row * p.ld + c;
        if (use && WIDE) {
            if (c < d) raw[r] = __ldg(reinterpret_cast<const uint4*>(src));
        } else if (use) {
            T* e = reinterpret_cast<T*>(&raw[r]);
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (c + j < d) e[j] = __ldg(src + j);
        }
    }
    float mx[R];
    unsigned most = 0u;
    bool bad[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const T* e = reinterpret_cast<const T*>(&raw[r]);
        mx[r] = 0.0f;
        bool b = false;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float v = fabsf(to_f32<T>(e[j]));
            b |= !(v <= FLT_MAX);
            mx[r] = fmaxf(mx[r], v);
        }
        bad[r] = __any_sync(0xffffffffu, b);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1)
#pragma unroll
        for (int r = 0; r < R; ++r) mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], o));
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = row0 + r;
        if (row >= p.n) break;
        const bool zero = bad[r] || !(mx[r] > 0.0f);
        const int e = zero ? 0 : max(-120, min(120, 13 - ilogbf(mx[r])));
        const float s = zero ? 0.0f : ldexpf(1.0f, e);
        const T* x = reinterpret_cast<const T*>(&raw[r]);
        __align__(16) __half hi[V], lo[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float v = zero ? 0.0f : to_f32<T>(x[j]) * s;
            hi[j] = __float2half_rn(v);
            lo[j] = __float2half_rn(v - __half2float(hi[j]));
        }
        __half* dst = p.out + (size_t)row * (size_t)(PARTS * kp) + c;
        if (c < kp) {
            if (V == 8) {
                *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(hi);
            } else {
                *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(hi);
                if (PARTS == 2)
                    *reinterpret_cast<uint2*>(dst + kp) = *reinterpret_cast<const uint2*>(lo);
            }
        }
        const float f = bad[r] ? __int_as_float(0x7fc00000) : zero ? 0.0f : ldexpf(1.0f, -e);
        if (lane == 0) p.f[row] = f;
        most = max(most, most_of(p, row, f));
    }
    return most;
}
// Both operands in one launch; the first block clears the error word.
template <typename T, int PARTS>
__global__ void __launch_bounds__(256)
    pack_kernel(const PackSide a, const PackSide b, int d, int kp, int* err) {
    if (err && blockIdx.x == 0 && threadIdx.x == 0) *err = 0;
    const bool first = (int)blockIdx.x < a.blocks;
    const PackSide& p = first ? a : b;
    if (p.seen || p.lse || p.weight) wait_for_last();  // (others: beside the kernel before it)
    const int row = (((int)blockIdx.x - (first ? 0 : a.blocks)) * 8 + (threadIdx.x >> 5)) * p.rows;
    const unsigned mine = row >= p.n      ? 0u
                          : p.rows != 4 ? pack_row<T, PARTS>(p, row, d, kp)
                          : p.wide      ? pack_short<T, PARTS, true>(p, row, d, kp)
                                        : pack_short<T, PARTS, false>(p, row, d, kp);
    wait_for_last();
    if (!p.largest) return;
    // the block's largest, unless it is there already
    __shared__ unsigned most[8];
    if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned m = 0;
        for (int i = 0; i < 8; ++i) m = max(m, most[i]);
        if (m > *(volatile unsigned*)p.largest) atomicMax(p.largest, m);
    }
}
// 16-bit rows copied to an aligned, zero-padded layout (their own is not one
// that a tensor map can describe).  A lane writes 16 bytes, from the five 32-bit
// words that hold them wherever the row starts; short rows share a warp.  Bound
// by memory: 209335 x 374 takes 50 us, its bytes 49.
__global__ void __launch_bounds__(256)
    align_kernel(const uint16_t* __restrict__ x, size_t ld, int n, int d, int kp, int shift,
                 uint16_t* __restrict__ out) {
    const int lanes = 1 << shift, lane = threadIdx.x & (lanes - 1);  // of a row
    const size_t row = ((size_t)blockIdx.x * 256 + threadIdx.x) >> shift;
    if (row >= (size_t)n) return;
    const uint16_t* src = x + row * ld;
    const int odd = (int)(reinterpret_cast<uintptr_t>(src) >> 1 & 1);
    // elements e and e + 1, which share a word; those outside of the row as zeros
    auto pair = [&](int e) -> uint32_t {
        const bool a = e >= 0 && e < d, b = e + 1 < d;
        if (a && b) return __ldg(reinterpret_cast<const uint32_t*>(src + e));
        return a ? (uint32_t)__ldg(src + e) : b ? (uint32_t)__ldg(src + e + 1) << 16 : 0u;
    };
    for (int c = lane * 8; c < kp; c += lanes * 8) {
        uint32_t w[5];
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = i < 4 || odd ? pair(c - odd + 2 * i) : 0u;
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = odd ? __byte_perm(w[i], w[i + 1], 0x5432) : w[i];
        *reinterpret_cast<uint4*>(out + row * kp + c) = make_uint4(v[0], v[1], v[2], v[3]);
    }
}
// ---------------------------------------------------------------------------
// the tensor-core pipeline
// ---------------------------------------------------------------------------
// STATS: running triples of 128 queries x one column tile of rows; GRAD: the
// score gradients of such a tile; PROD_Q, PROD_X: the products of the score
// gradients with the rows and (transposed) with the queries.
constexpr int STATS = 0, GRAD = 1, PROD_Q = 2, PROD_X = 3;

struct Mma {
    // Units: STATS, GRAD: (row block, chunk of the column tiles), the row
    // block fastest so that the blocks that run together share column tiles.
    // PROD: (row block, column block, split of K).
    int mt, nt, chunks;
    int atoms;                   // 64-wide steps of K
    int klast;                   // 16-wide MMA steps of the last of them
    int resident;                // STATS, GRAD: A's K steps stay in shared memory for a unit
    int a_part, b_part;          // distance of the second part from the first in its map
    int b_row0;                  // PROD_Q: first row of the chunk
    int ncols;                   // PROD: columns of the output
    uint32_t idesc;              // but for N
    int stall;                   // test hook: no loads, so that the waits run out
    int* err;
    unsigned long long wait;
};
struct StatsArgs {
    int q0, nq;                 // queries [q0, q0 + nq) of the call
    int n;
    const float* qf;            // [nq] 2^-e of the packed queries (f32 rows), else null
    const float* xf;            // [padded n] 2^-e of the packed rows, else null
    float rf;                   // scale * log2(e)
    const uint32_t* allowed;    // nullable
    size_t ld_allowed;          // words a query (0: one filter for all)
    float4* part;               // [chunks * 4][nq]: m, l, a (see Run)
    float2* top;                // [nq][groups] or null, in units of t
    size_t groups;              // 32-row groups, whole column tiles
    float* size;                // [blocks] largest xf, with f32 rows and top
};
// What the score gradients of one query need (see coef_of).
struct Coef {
    float rf_hi, rf_lo, l_hi, l_lo;  // t - lse in log2 units = u rf - l, in two parts each
    float c, h, g;                   // G W = p (c + h x) + g at the given row
    int target;
};
// The head of the gradient's workspace, cleared by head_kernel.
struct GradHead {
    unsigned q_most;            // WEIGHT_ZERO + the largest exponent of qf_i B_i
    float x_most;               // the largest xf
};
struct GradArgs {
    int nq, n, j0, cols;        // this chunk: rows [j0, j0 + cols)
    const Coef* coef;           // [nq]
    const float* xf;            // 2^-e of the packed rows, over the largest
    const uint32_t* allowed;
    size_t ld_allowed;
    size_t ldg;                 // output [parts][nqp][ldg]
    int nqp;
    float* rest;                // one part: [nq] what fp16 leaves of the given row's G
};
struct ProdArgs {
    int rows, cols;             // output
    const float* f;             // see out_factor
    const GradHead* head;
    float* partial;             // [splits][rows][cols], or null: `out` is written
    int add;                    // added to `partial` instead of stored
    void* out;
    size_t ldo;
    int dtype;
};

// What an output row is multiplied with: of the queries (no head) its own factor
// f, of the rows 2^(most - 13) / f.  (See settle_kernel.)
__device__ __forceinline__ float out_factor(float f, const GradHead* head) {
    if (!head) return f;
    return ldexpf(1.0f / f, min((int)head->q_most - WEIGHT_ZERO - 13, 120));
}

__device__ __forceinline__ uint32_t allowed_word(const uint32_t* al, size_t ld, int q, size_t col,
                                                 int n) {
    if (col >= (size_t)n) return 0u;
    const uint32_t w = al ? __ldg(al + (size_t)q * ld + (col >> 5)) : 0xffffffffu;
    const size_t left = (size_t)n - col;
    return left >= 32 ? w : w & ((1u << left) - 1u);
}

// One 32-column chunk of the accumulator, in f32.
__device__ __forceinline__ void load_chunk(uint32_t tmem, float (&u)[32]) {
    uint32_t v[32];
    tmem_ld32_nowait(tmem, v);
    tmem_wait_regs(v);
#pragma unroll
    for (int i = 0; i < 32; ++i) u[i] = __uint_as_float(v[i]);
}
// ---- pairs of blocks ----
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// The address, in the cluster's window, of the first block's copy of `p`.
__device__ __forceinline__ uint32_t leader_addr(const void* p) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Into this block's shared memory, counted on the first block's barrier.
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, uint32_t bar,
                                              int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
        : "memory");
}
__device__ __forceinline__ void tma_store(const void* src, const CUtensorMap* map, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
            reinterpret_cast<uint64_t>(map)),
        "r"(smem_u32(src)), "r"(x), "r"(y)
        : "memory");
}
__device__ __forceinline__ void umma_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                          uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
// Arrives on the barrier of both blocks when the MMAs issued so far are done.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}
// One lane of a converged warp.  The issuing warps stay converged and only
// this lane issues: the copies and MMAs take their operands from uniform
// registers, which a branch on the lane number would have to fill lane by
// lane (measured, 2048 x 131072 x 768 bf16: 424 us instead of 295).
__device__ __forceinline__ bool elected() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(p));
    return p != 0;
}
// A bounded wait of a whole converged warp.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err,
                                          unsigned long long limit) {
    return __all_sync(0xffffffffu, mbar_wait_spin(bar, parity, err, limit));
}
// Tells the first block that an accumulator was read.  Relaxed: the barrier
// hands over tensor memory alone, and tcgen05.wait::ld, before it, has returned
// only when the values were in registers.  A release would first wait for the
// thread's stores to reach L2, the groups' largest scores of the tile before
// (4096 x 262144 x 96 f32, k = 10: 1152 us instead of 811).
__device__ __forceinline__ void arrive_leader(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
                 : "memory");
}

// What a chunk of 32 columns needs besides its scores: the filter's word of
// the thread's row, and (scaled rows) the columns' factors, in the warp's own
// shared memory.  `load` starts the reads of a tile's chunks while the tile
// before it is worked on, `ready` hands them over.  BIAS, with a filter that all
// queries share: what it adds to the columns (0 or NONE) lies there too, one
// packed addition for two columns instead of a test and a select for each (the
// factor of a column that nobody may see is 0, whatever its row holds).
template <bool FACTORS, bool BIAS, int CHUNKS>
struct Columns {
    uint32_t next[CHUNKS], word[CHUNKS];
    float nf[CHUNKS];
    float* fac;  // [CHUNKS][32], then the biases
    bool shared_filter;
    __device__ __forceinline__ void load(const uint32_t* al, const float* f, size_t col, int n) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int h = 0; h < CHUNKS; ++h) {
            next[h] = allowed_word(al, 0, 0, col + 32 * h, n);
            if (FACTORS) nf[h] = __ldg(f + col + 32 * h + lane);
        }
    }
    __device__ __forceinline__ void ready() {
        if (FACTORS || BIAS) __syncwarp();
#pragma unroll
        for (int h = 0; h < CHUNKS; ++h) {
            word[h] = next[h];
            const int lane = threadIdx.x & 31;
            const bool out = BIAS && shared_filter && !(next[h] >> lane & 1u);
            if (FACTORS) fac[32 * h + lane] = out ? 0.0f : nf[h];
            if (BIAS) fac[32 * (CHUNKS + h) + lane] = out ? NONE : 0.0f;
        }
        if (FACTORS || BIAS) __syncwarp();
    }
};

// The epilogues: one object per thread and unit; `chunk` takes 32 columns of
// the thread's row, from column `col` of the unit's matrix (chunk h of the
// thread's columns of the tile), in registers.
template <bool TWO, bool BLK>
struct StatsEpilogue {
    typedef StatsArgs Args;
    const StatsArgs& p;
    int q;  // query of this pass, -1 past the end
    float rf;
    Run r;
    bool live;
    Columns<TWO, TWO, BLK ? 1 : 2> c;
    const uint32_t* al;
    float top_max;  // largest group's score of the unit (unmarked)
    __device__ StatsEpilogue(const StatsArgs& a, int row, int row0, int, float* fac,
                             unsigned char*, const CUtensorMap*)
        : p(a) {
        c.fac = fac;
        c.shared_filter = a.ld_allowed == 0;
        q = row < a.nq ? row : -1;
        // (with a filter of its own, rows past the end see everything: never stored)
        al = !a.allowed || (q < 0 && a.ld_allowed)
                 ? nullptr
                 : a.allowed + (size_t)(a.q0 + max(q, 0)) * a.ld_allowed;
        live = row0 < a.nq;
        rf = a.rf;
        if (TWO && q >= 0) {
            const float f = a.qf[q];
            rf = f == 0.0f ? a.rf : f * a.rf;  // a query of zeros scores 0
        }
        r = run_empty();
        top_max = NONE;
    }
    __device__ __forceinline__ void load(int col) { c.load(al, p.xf, (size_t)col, p.n); }
    // SEEN: 0: all rows see all columns; 1: each by its own word; 2: all rows
    // see the same, by the columns' biases.  Copies of the code, as the selects
    // are not free.
    template <int SEEN>
    __device__ __forceinline__ float2 fold(const float (&u)[32], uint32_t w, int h) {
        constexpr int BIAS_AT = 32 * (BLK ? 1 : 2);
        const float4* bias = reinterpret_cast<const float4*>(c.fac + BIAS_AT + 32 * h);
        const float4* fac = reinterpret_cast<const float4*>(c.fac + 32 * h);
        const uint64_t rf2 = packf(rf, rf), nm2 = packf(-r.m, -r.m);
        float d[32];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint64_t t0 = packf(u[4 * i], u[4 * i + 1]), t1 = packf(u[4 * i + 2], u[4 * i + 3]);
            if (TWO) {
                const float4 f = fac[i];
                t0 = mul2(t0, packf(f.x, f.y));
                t1 = mul2(t1, packf(f.z, f.w));
            }
            t0 = fma2(t0, rf2, nm2);
            t1 = fma2(t1, rf2, nm2);
            if (SEEN == 2) {
                const float4 f = bias[i];
                t0 = add2(t0, packf(f.x, f.y));
                t1 = add2(t1, packf(f.z, f.w));
            }
            d[4 * i] = lo_of(t0);
            d[4 * i + 1] = hi_of(t0);
            d[4 * i + 2] = lo_of(t1);
            d[4 * i + 3] = hi_of(t1);
        }
        if (SEEN == 1) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (!(w >> i & 1u)) d[i] = NONE;
        }
        float2 best = make_float2(NONE, NONE);
        float cm;
        if (p.top) {
            best = top_pair(d);
            // (the mark may have moved it; by far less than RAISE)
            cm = best.x;
            if (best.x > NONE_BELOW) {
                const float v = unmarked(unmarked(best.x) + r.m);
                best.x = __uint_as_float(__float_as_uint(v) | (__float_as_uint(best.x) & 15u));
                top_max = fmaxf(top_max, v);
            }
            best.y += r.m;
        } else {
            cm = max3(d[0], d[1], d[2]);
#pragma unroll
            for (int i = 3; i < 31; i += 2) cm = max3(cm, d[i], d[i + 1]);
            cm = fmaxf(cm, d[31]);
        }
        if (cm > r.limit) {
            const float by = run_raise(r, cm);
#pragma unroll
            for (int i = 0; i < 32; ++i) d[i] -= by;
        }
        uint64_t l2[2] = {0, 0}, a2[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint64_t e = packf(ex2(d[2 * i]), ex2(d[2 * i + 1]));
            l2[i & 1] = add2(l2[i & 1], e);
            a2[i & 1] = fma2(e, packf(d[2 * i], d[2 * i + 1]), a2[i & 1]);
        }
        l2[0] = add2(l2[0], l2[1]);
        a2[0] = add2(a2[0], a2[1]);
        r.l += lo_of(l2[0]) + hi_of(l2[0]);
        r.a += lo_of(a2[0]) + hi_of(a2[0]);
        return best;
    }
    __device__ __forceinline__ void chunk(float (&u)[32], int icol, int h) {
        if (!live) return;
        const size_t col = (size_t)icol;
        const uint32_t w = h ? c.word[sizeof(c.word) / 4 - 1] : c.word[0];
        float2 best = make_float2(NONE, NONE);
        if (__all_sync(0xffffffffu, w == 0xffffffffu)) best = fold<0>(u, w, h);
        else if (__any_sync(0xffffffffu, w != 0u))
            best = TWO && c.shared_filter ? fold<2>(u, w, h) : fold<1>(u, w, h);
        if (p.top && q >= 0) p.top[(size_t)q * p.groups + (col >> 5)] = best;
    }
    __device__ __forceinline__ void finish(int chunk, int part) {
        if (q >= 0) p.part[(size_t)(chunk * 4 + part) * p.nq + q] = run_stored(r, top_max);
    }
};

// Score gradients, stored as fp16 (two parts for f32 inputs) scaled by 2^-ej and
// the query's W (see settle_kernel) so that both products read them as they are.
// One part rounds G by up to 2^-11 of it, as a result in f16 is rounded and an
// eighth of what a bf16 one is; a second part would cost a second product each.
// (d_queries gets back what is cut off the given row's G, d_rows does not: it would
// take a sum over the queries that share a given row.  Of 601 x 30011 x 200 f16 d_rows is off
// by 2.9e-4 of its norm, its own rounding is 2.1e-4; of some ten queries by up to 4.2e-4.)
template <bool TWO, bool BLK>
struct GradEpilogue {
    typedef GradArgs Args;
    const GradArgs& p;
    int q, row;
    bool live;  // (rows up to a multiple of 128 are written)
    Coef k;
    Columns<true, false, BLK ? 1 : 2> c;
    const uint32_t* al;
    unsigned char* stage;      // the warp's staged outputs, part 1 STAGED bytes on
    const CUtensorMap* omap;
    __device__ GradEpilogue(const GradArgs& a, int r, int row0, int, float* fac,
                            unsigned char* staged, const CUtensorMap* out)
        : p(a), stage(staged), omap(out) {
        live = row0 < (a.nq + BM - 1) / BM * BM;
        c.fac = fac;
        row = r;
        al = r >= a.nq || !a.allowed ? nullptr : a.allowed + (size_t)r * a.ld_allowed;
        q = r < a.nq ? r : -1;
        // (a row past the last query has no given row: it would leave the rest of
        // its rounding in front of p.rest)
        k = Coef{};
        k.target = -1;
        if (q >= 0) k = a.coef[q];
    }
    __device__ __forceinline__ void load(int col) {
        c.load(al, p.xf, (size_t)p.j0 + col, p.j0 + p.cols);
    }
    __device__ __forceinline__ void chunk(float (&u)[32], int icol, int h) {
        const size_t col = (size_t)icol, gcol = (size_t)p.j0 + col;
        if (col >= p.ldg || !live) return;
        const uint32_t w = q < 0 ? 0u : h ? c.word[sizeof(c.word) / 4 - 1] : c.word[0];
        if (!__any_sync(0xffffffffu, w != 0u)) {
#pragma unroll
            for (int i = 0; i < 32; ++i) u[i] = 0.0f;
            store(u, col);
            return;
        }
        const uint64_t rh2 = packf(k.rf_hi, k.rf_hi), rl2 = packf(k.rf_lo, k.rf_lo);
        const uint64_t lh2 = packf(-k.l_hi, -k.l_hi), ll2 = packf(-k.l_lo, -k.l_lo);
        const uint64_t h2 = packf(k.h, k.h), c2 = packf(k.c, k.c);
        const float2* xf = reinterpret_cast<const float2*>(c.fac + 32 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float2 f = xf[i];
            const uint64_t f2 = packf(f.x, f.y);
            const uint64_t t = mul2(packf(u[2 * i], u[2 * i + 1]), f2);
            const uint64_t y = add2(fma2(t, rh2, lh2), fma2(t, rl2, ll2));
            const float x0 = fmaxf(lo_of(y), -160.0f), x1 = fmaxf(hi_of(y), -160.0f);
            uint64_t g = mul2(packf(ex2(x0), ex2(x1)), fma2(packf(x0, x1), h2, c2));
            g = mul2(g, f2);
            u[2 * i] = lo_of(g);
            u[2 * i + 1] = hi_of(g);
        }
        const int at = k.target - (int)gcol;  // of the given row, if it is in this chunk
        if ((unsigned)at < 32u) {
            const float add = k.g * c.fac[32 * h + at];
            float all = 0.0f;
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (i == at) all = u[i] += add;
            // the largest G of most queries: what its rounding leaves is added to
            // d_queries on its own (else it is most of the error of f16 results)
            if (!TWO) p.rest[q] = all - __half2float(__float2half_rn(all));
        }
        __syncwarp();
        if (!__all_sync(0xffffffffu, w == 0xffffffffu)) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (!(w >> i & 1u)) u[i] = 0.0f;
        }
        store(u, col);
    }
    // The warp's 32 x 32 values, staged in rows of 64 bytes (64-byte swizzle:
    // 16-byte piece b of row r at b ^ (r / 2 % 4), so that eight lanes' pieces
    // lie in different banks) and stored by TMA: straight from registers each
    // 16-byte store of a warp would touch 32 lines (measured at 4096 x 65536:
    // 120 us of 440).
    __device__ __forceinline__ void store(const float (&u)[32], size_t col) {
        const int lane = threadIdx.x & 31;
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
        unsigned char* o = stage + lane * 64;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            uint32_t h4[4], l4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float g0 = u[8 * b + 2 * i], g1 = u[8 * b + 2 * i + 1];
                const __half2 hh = __floats2half2_rn(g0, g1);
                h4[i] = *reinterpret_cast<const uint32_t*>(&hh);
                if (TWO) {
                    const float2 back = __half22float2(hh);
                    const __half2 ll = __floats2half2_rn(g0 - back.x, g1 - back.y);
                    l4[i] = *reinterpret_cast<const uint32_t*>(&ll);
                }
            }
            const int at = 16 * (b ^ (lane >> 1 & 3));
            *reinterpret_cast<uint4*>(o + at) = make_uint4(h4[0], h4[1], h4[2], h4[3]);
            if (TWO)
                *reinterpret_cast<uint4*>(o + STAGED + at) = make_uint4(l4[0], l4[1], l4[2], l4[3]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
            const int y = row;  // (lane 0: the warp's first row)
            tma_store(stage, omap, (int)col, y);
            if (TWO) tma_store(stage + STAGED, omap, (int)col, p.nqp + y);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
    }
    __device__ __forceinline__ void finish(int, int) {
        if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
};

// Transposes a warp's 32 x 32 values: lane i's v[j] goes to lane j's v[i].
__device__ __forceinline__ void transpose32(float (&v)[32]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int s = 16; s; s >>= 1) {
        const bool up = lane & s;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            if (i & s) continue;
            const float give = up ? v[i] : v[i | s];
            const float got = __shfl_xor_sync(0xffffffffu, give, s);
            if (up) v[i] = got;
            else v[i | s] = got;
        }
    }
}
__device__ __forceinline__ void put(void* out, size_t o, int dtype, float v) {
    if (dtype == FDB_DTYPE_F32) static_cast<float*>(out)[o] = v;
    else if (dtype == FDB_DTYPE_BF16) static_cast<__nv_bfloat16*>(out)[o] = __float2bfloat16_rn(v);
    else static_cast<__half*>(out)[o] = __float2half_rn(v);
}

// Stores go a row at a time, its 32 columns by the warp's lanes (whatever the
// rows' alignment): a thread's own row in 16-byte pieces would touch 32 lines
// an instruction.
struct ProdEpilogue {
    typedef ProdArgs Args;
    const ProdArgs& p;
    int row, row0, split;
    float s;
    Columns<false, false, 1> c;
    __device__ ProdEpilogue(const ProdArgs& a, int r, int r0, int sp, float*, unsigned char*,
                            const CUtensorMap*)
        : p(a) {
        row = r;
        row0 = r0;
        split = sp;
        s = !a.partial && row < a.rows ? out_factor(a.f[row], a.head) : 0.0f;
    }
    __device__ __forceinline__ void load(int) {
        c.next[0] = 0;
    }
    __device__ __forceinline__ void chunk(float (&u)[32], int c, int) {
        if (c >= p.cols || row0 >= p.rows) return;
        const int lane = threadIdx.x & 31, rows = min(32, p.rows - row0);
        if (!p.partial) {
#pragma unroll
            for (int i = 0; i < 32; ++i) u[i] *= s;
        }
        transpose32(u);
        if (c + lane >= p.cols) return;
        if (!p.partial) {
            size_t o = (size_t)row0 * p.ldo + c + lane;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                if (i < rows) put(p.out, o, p.dtype, u[i]);
                o += p.ldo;
            }
            return;
        }
        float* o = p.partial + ((size_t)split * p.rows + row0) * (size_t)p.cols + c + lane;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            if (i < rows) *o = p.add ? *o + u[i] : u[i];
            o += p.cols;
        }
    }
    __device__ __forceinline__ void finish(int, int) {}
};
template <int MODE, bool TWO, bool BLK>
struct EpilogueOf;
template <bool TWO, bool BLK>
struct EpilogueOf<STATS, TWO, BLK> {
    typedef StatsEpilogue<TWO, BLK> Type;
};
template <bool TWO, bool BLK>
struct EpilogueOf<GRAD, TWO, BLK> {
    typedef GradEpilogue<TWO, BLK> Type;
};
template <bool TWO>
struct EpilogueOf<PROD_Q, TWO, TWO> {
    typedef ProdEpilogue Type;
};
template <bool TWO>
struct EpilogueOf<PROD_X, TWO, TWO> {
    typedef ProdEpilogue Type;
};

// MN-major operand tile (64 elements of M or N along a 128-byte row, one row
// a k, 128-byte swizzle): 8-k groups 1024 B apart (SBO), 64-element groups
// 64 k = 8192 B apart (LBO).
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)512 << 16) | ((uint64_t)64 << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// What a unit covers.
struct Unit {
    int mt, sp;      // sp: chunk (STATS, GRAD) or split of K (PROD)
    int t0, t1;      // column tiles
    int a0, a1;      // 64-wide steps of K
};
template <int MODE>
__device__ __forceinline__ Unit unit_of(const Mma& g, int u) {
    Unit x;
    x.mt = u % g.mt;
    if (MODE == PROD_Q || MODE == PROD_X) {
        x.t0 = u / g.mt % g.nt;
        if (MODE == PROD_X) {  // the large operand's rows once for all column tiles
            x.t0 = u % g.nt;
            x.mt = u / g.nt % g.mt;
        }
        x.t1 = x.t0 + 1;
        x.sp = u / (g.mt * g.nt);
        x.a0 = (int)((long long)x.sp * g.atoms / g.chunks);
        x.a1 = (int)((long long)(x.sp + 1) * g.atoms / g.chunks);
    } else {
        x.sp = u / g.mt;
        x.t0 = (int)((long long)x.sp * g.nt / g.chunks);
        x.t1 = (int)((long long)(x.sp + 1) * g.nt / g.chunks);
        x.a0 = 0;
        x.a1 = g.atoms;
    }
    return x;
}

// A pair of blocks works on 256 rows x one column tile.  In each, warp 0 loads
// its share of the K steps with TMA and sixteen epilogue warps (four per lane
// quadrant, a quarter of the columns each) work on the block's 128 rows of a
// finished accumulator; warp 1 of the first block issues the MMAs of both.
// Persistent: a pair takes units blockIdx.x / 2, + gridDim.x / 2, ...
//
// The tensor core's own additions cut a sum towards zero, once for 16 of K:
// measured on one row, a score comes out short by 4e-8 of itself for each 32
// of K (bf16; f16, whose products have more bits to cut, up to 1.3e-7).  Where
// that matters (f32, and long rows) sums are taken in blocks (BLK): an
// accumulator holds 128 of K (TWO parts: first the products lo.hi and hi.lo,
// then hi.hi) or 256, and the epilogue adds them up in registers.  Else an
// accumulator is a whole tile.  GRAD takes 64 of K of two parts, whose sums it has
// the time for: what a score is off by, its probability is off by of itself (d_rows of
// 125 x 4405 x 74 f32: 1.3e-6 of its norm with 128, 4.6e-7 with 64 and the half
// of cut_of; 60 us either way).
template <int MODE, bool TWO, bool BLK>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    rows_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap,
                const __grid_constant__ CUtensorMap omap, const Mma g,
                const typename EpilogueOf<MODE, TWO, BLK>::Type::Args p) {
    constexpr bool PROD = MODE == PROD_Q || MODE == PROD_X;
    constexpr bool A_MN = MODE == PROD_X, B_MN = PROD;
    constexpr int BN = bn_of(BLK), NST = stages_of(TWO, BLK, MODE == GRAD), NACC = accs_of(BLK);
    constexpr int STAGE = stage_bytes(TWO, BLK), PARTS = TWO ? 2 : 1;
    constexpr int KBLOCK = kblock_of(TWO, MODE == GRAD);
    constexpr int B0 = PARTS * OPER;               // operand B in a stage
    constexpr int B_PART = BN / 2 * 128;           // bytes of one part of this block's half
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const uint32_t base = smem_u32(smem_raw);
    unsigned char* smem = smem_raw + ((1024 - (base & 1023)) & 1023);
    constexpr int RING = NST * STAGE;
    unsigned char* staged = smem + RING;
    unsigned char* after = staged + staged_of(TWO, MODE == GRAD);
    // Few K steps: all of A at the ring's start, and stages of B alone.
    const bool resident = !PROD && g.resident;
    const int a_bytes = resident ? g.atoms * PARTS * OPER : 0;
    const int stage = resident ? PARTS * B_PART : STAGE;
    const int nst = resident ? min(MAX_STG, (RING - a_bytes) / stage) : NST;
    const int b_at = resident ? 0 : B0;
    unsigned char* ring = smem + a_bytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(after);               // the first block's count
    uint64_t* empty = full + MAX_STG;
    uint64_t* t_full = empty + MAX_STG;
    uint64_t* t_empty = t_full + NACC;                                 // the first block's count
    uint64_t* a_full = t_empty + NACC;                                 // the first block's counts
    uint64_t* a_empty = a_full + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(a_empty + 1);
    float* factors = reinterpret_cast<float*>(after + 256);             // [16 warps][128]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const uint32_t full0 = leader_addr(full);
    if (threadIdx.x == 0) {
        for (int i = 0; i < MAX_STG; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < NACC; ++i) {
            mbar_init(t_full + i, 1);
            mbar_init(t_empty + i, 2 * EPI_WARPS);
        }
        mbar_init(a_full, 1);
        mbar_init(a_empty, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(tmem_slot)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        tc_fence_before();
    }
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    wait_for_last();
    const int units = PROD ? g.mt * g.nt * g.chunks : g.mt * g.chunks;
    int last_stage = -1;  // MMA issuer: last stage committed, and its phase
    uint32_t last_phase = 0;

    if (warp == 0) {
        int s = 0, use = 0, ui = 0;  // stage, how often it was used before, units
        bool ok = !g.stall;
        for (int u = pair; ok && u < units; u += pairs, ++ui) {
            const Unit x = unit_of<MODE>(g, u);
            const int m0 = x.mt * PM + rank * BM;
            if (resident) {
                if (ui > 0 && !warp_wait(a_empty, (ui - 1) & 1, g.err, g.wait)) break;
                if (elected()) {
                    if (rank == 0) mbar_expect_tx(a_full, 2 * (uint32_t)a_bytes);
                    const uint32_t bar = leader_addr(a_full);
                    for (int a = 0; a < g.atoms; ++a)
#pragma unroll
                        for (int h = 0; h < PARTS; ++h)
                            tma_load_pair(smem + (a * PARTS + h) * OPER, &amap, bar,
                                          h * g.a_part + a * KATOM, m0);
                }
                __syncwarp();
            }
            for (int t = x.t0; ok && t < x.t1; ++t) {
                // this block's half of the columns: [n0, n0 + half)
                const int half = PROD ? ((min(BN, g.ncols - t * BN) + 31) & ~31) / 2 : BN / 2;
                const int n0 = t * BN + rank * half;
                const int boxes = B_MN ? (half + 63) / 64 : 0;
                const uint32_t bytes =
                    PARTS * ((resident ? 0 : OPER) + (uint32_t)(B_MN ? boxes * 8192 : B_PART));
                for (int a = x.a0; a < x.a1; ++a) {
                    if (use > 0 && !warp_wait(empty + s, (use - 1) & 1, g.err, g.wait)) {
                        ok = false;
                        break;
                    }
                    if (elected()) {
                        if (rank == 0) mbar_expect_tx(full + s, 2 * bytes);
                        const uint32_t bar = full0 + 8 * s;
#pragma unroll
                        for (int h = 0; h < PARTS; ++h) {
                            unsigned char* da = ring + s * stage + h * OPER;
                            unsigned char* db = ring + s * stage + b_at + h * B_PART;
                            const int pa = h * g.a_part, pb = h * g.b_part;
                            if (resident) {
                            } else if (A_MN) {
                                tma_load_pair(da, &amap, bar, m0, pa + a * KATOM);
                                tma_load_pair(da + 8192, &amap, bar, m0 + 64, pa + a * KATOM);
                            } else if (PROD) {
                                tma_load_pair(da, &amap, bar, a * KATOM, pa + m0);
                            } else {
                                tma_load_pair(da, &amap, bar, pa + a * KATOM, m0);
                            }
                            if (B_MN) {
                                tma_load_pair(db, &bmap, bar, pb + n0, g.b_row0 + a * KATOM);
                                if (boxes > 1)
                                    tma_load_pair(db + 8192, &bmap, bar, pb + n0 + 64,
                                                  g.b_row0 + a * KATOM);
                            } else {
                                tma_load_pair(db, &bmap, bar, pb + a * KATOM, g.b_row0 + n0);
                            }
                        }
                    }
                    __syncwarp();
                    if (++s == nst) s = 0, ++use;
                }
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            int s = 0, ti = 0, ui = 0;  // stage, accumulators, units
            uint32_t phase = 0;         // of the stage
            bool ok = true;
            for (int u = pair; ok && u < units; u += pairs, ++ui) {
                const Unit x = unit_of<MODE>(g, u);
                if (resident && !warp_wait(a_full, ui & 1, g.err, g.wait)) break;
                for (int t = x.t0; ok && t < x.t1; ++t) {
                    const int bn = PROD ? (min(BN, g.ncols - t * BN) + 31) & ~31 : BN;
                    const uint32_t idesc = g.idesc | ((uint32_t)(bn >> 3) << 17);
                    for (int a = x.a0; ok && a < x.a1;) {
                        // an accumulator: KBLOCK steps, or all
                        const int b = ti % NACC;
                        const int a1 = BLK ? min(x.a1, a + KBLOCK) : x.a1;
                        const uint32_t d = tmem + (uint32_t)(b * BN);
                        if (ti >= NACC &&
                            !warp_wait(t_empty + b, (ti / NACC - 1) & 1, g.err, g.wait)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        // (past the operands' last column the steps hold zeros)
                        auto issue = [&](int slot, int atom, int ao, int bo, bool first) {
                            const uint32_t sp = smem_u32(ring + slot * stage);
                            const uint32_t ap =
                                (resident ? smem_u32(smem + atom * PARTS * OPER) : sp) + ao;
                            const uint32_t bp = sp + b_at + bo;
                            const int kk1 = atom == g.atoms - 1 ? g.klast : 4;
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)
                                if (kk < kk1)
                                    umma_pair(d,
                                              A_MN ? smem_desc_mn(ap + kk * 2048)
                                                   : smem_desc_sw128(ap + kk * 32),
                                              B_MN ? smem_desc_mn(bp + kk * 2048)
                                                   : smem_desc_sw128(bp + kk * 32),
                                              idesc, !first || kk > 0);
                        };
                        const int s0 = s, from = a;
                        uint32_t last = 0;
                        for (; a < a1; ++a) {
                            if (!warp_wait(full + s, phase, g.err, g.wait)) {
                                ok = false;
                                break;
                            }
                            tc_fence_after();
                            if (elected()) {
                                if (TWO) {
                                    issue(s, a, OPER, 0, a == from);
                                    issue(s, a, 0, B_PART, false);
                                } else {
                                    issue(s, a, 0, 0, a == from);
                                    umma_commit_pair(empty + s);
                                    if (a + 1 == a1) umma_commit_pair(t_full + b);
                                }
                            }
                            __syncwarp();
                            if (!TWO) last_stage = s, last_phase = phase;
                            else last = phase;
                            if (++s == nst) s = 0, phase ^= 1;
                        }
                        if (TWO && ok) {
                            int i = s0;
                            for (int atom = from; atom < a1; ++atom) {
                                if (elected()) {
                                    issue(i, atom, 0, 0, false);
                                    umma_commit_pair(empty + i);
                                    if (atom + 1 == a1) umma_commit_pair(t_full + b);
                                }
                                __syncwarp();
                                last_stage = i;
                                if (++i == nst) i = 0;
                            }
                            last_phase = last;
                        }
                        ++ti;
                    }
                }
                if (resident && ok) {
                    if (elected()) umma_commit_pair(a_empty);
                    __syncwarp();
                }
            }
        }
    } else if (warp == 2) {
        // (else idle) the largest factor of the rows that a shared filter lets see,
        // all rows with filters of their own
        if constexpr (MODE == STATS && TWO) {
            if (p.size) {
                const uint32_t* al = p.ld_allowed ? nullptr : p.allowed;
                float m = 0.0f;
                for (int j = blockIdx.x * 32 + lane; j < p.n; j += gridDim.x * 32)
                    if (!al || (__ldg(al + (j >> 5)) >> lane & 1u)) m = fmaxf(m, p.xf[j]);
                const int most = __reduce_max_sync(0xffffffffu, __float_as_int(m));
                if (lane == 0) p.size[blockIdx.x] = __int_as_float(most);
            }
        }
    } else if (warp >= EPI_WARP0) {
        const int w = warp - EPI_WARP0, quad = w & 3, part = w >> 2;
        const uint32_t mine = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(part * (BN / 4));
        const uint32_t release0 = leader_addr(t_empty);
        int ti = 0;
        bool ok = true;
        // the next accumulator, or false when the kernel is aborting
        auto next = [&]() -> bool {
            int got = 0;
            if (lane == 0) got = mbar_wait_spin(t_full + ti % NACC, (ti / NACC) & 1, g.err, g.wait);
            got = __shfl_sync(0xffffffffu, got, 0);
            tc_fence_after();
            return got != 0;
        };
        auto release = [&] {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_leader(release0 + 8 * (ti % NACC));
            ++ti;
        };
        for (int u = pair; ok && u < units; u += pairs) {
            const Unit x = unit_of<MODE>(g, u);
            const int row0 = x.mt * PM + rank * BM + quad * 32;
            typename EpilogueOf<MODE, TWO, BLK>::Type epi(
                p, row0 + lane, row0, x.sp, factors + w * 128,
                staged + (MODE == GRAD ? w * PARTS * STAGED : 0), &omap);
            epi.load(x.t0 * BN + part * (BN / 4));
            for (int t = x.t0; ok && t < x.t1; ++t) {
                const int col = t * BN + part * (BN / 4);
                epi.c.ready();
                if (t + 1 < x.t1) epi.load(col + BN);
                float v[32];
                if (BLK) {
                    if (!next()) {
                        ok = false;
                        break;
                    }
                    load_chunk(mine + (uint32_t)(ti % NACC * BN), v);
                    release();
                    for (int a = x.a0 + KBLOCK; a < x.a1; a += KBLOCK) {
                        if (!next()) {
                            ok = false;
                            break;
                        }
                        float y[32];
                        load_chunk(mine + (uint32_t)(ti % NACC * BN), y);
                        release();
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] += y[i];
                    }
                    if (ok) epi.chunk(v, col, 0);
                    __syncwarp();
                } else {
                    if (!next()) {
                        ok = false;
                        break;
                    }
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        load_chunk(mine + (uint32_t)(ti % NACC * BN + h * 32), v);
                        epi.chunk(v, col + h * 32, h);
                        __syncwarp();
                    }
                    release();
                }
            }
            if (ok) epi.finish(x.sp, part);
        }
    }
    // One verdict for the block.  An aborting block gives the copies that it
    // issued (which the first block's barriers count, so they cannot be waited
    // for here) time to land, and the MMAs; then the pair leaves together.
    if (__syncthreads_or(*(volatile int*)g.err != 0)) {
        const unsigned long long c0 = clock64();
        if (warp == 0)
            while (clock64() - c0 < DRAIN_CYCLES) __nanosleep(1000);
        if (warp == 1 && lane == 0 && last_stage >= 0)
            while (!mbar_try(empty + last_stage, last_phase) && clock64() - c0 < DRAIN_CYCLES) {
            }
        if (MODE == GRAD && warp >= EPI_WARP0 && lane == 0)
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncthreads();
    }
    cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                     "r"(512));
    }
}

__device__ __forceinline__ __half2 pair_twice(__half x) { return __half2half2(x); }
__device__ __forceinline__ __nv_bfloat162 pair_twice(__nv_bfloat16 x) {
    return __bfloat162bfloat162(x);
}
// The largest size of the elements that a thread has read.
template <typename T>
struct Largest {
    using Pair = decltype(pair_twice(T()));
    Pair m = pair_twice(T(0.0f));
    __device__ __forceinline__ void add(const uint4& raw) {
        const Pair* e = reinterpret_cast<const Pair*>(&raw);
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __hmax2(m, __habs2(e[i]));
    }
    __device__ __forceinline__ void add(T x) { m = __hmax2(m, __habs2(pair_twice(x))); }
    __device__ __forceinline__ float get() const {
        return fmaxf(to_f32<T>(m.x), to_f32<T>(m.y));
    }
};
template <>
struct Largest<float> {
    float m = 0.0f;
    __device__ __forceinline__ void add(const uint4& raw) {
        m = max3(m, fabsf(__uint_as_float(raw.x)), fabsf(__uint_as_float(raw.y)));
        m = max3(m, fabsf(__uint_as_float(raw.z)), fabsf(__uint_as_float(raw.w)));
    }
    __device__ __forceinline__ void add(float x) { m = fmaxf(m, fabsf(x)); }
    __device__ __forceinline__ float get() const { return m; }
};
// ---------------------------------------------------------------------------
// a few queries: one pass over the rows on the FMA pipes
// ---------------------------------------------------------------------------
// A warp takes groups of 32 rows, RB at a time: each lane multiplies its
// columns of RB rows with its columns of NQ queries (from shared memory, two
// products an instruction), and a transposing reduction leaves each row's sums
// in 32 / RB lanes, of which one keeps them, so that after all batches every
// lane holds one row of the group.  Bound by memory (each row read once) up to
// about 8 queries; the tensor cores would work on 256 rows of queries.
// TOP, with alternatives: finds the largest element of the rows that some query
// sees, too (up to 7 % of the time: 100000 x 768 f32, 4 queries, 113 -> 120 us).
// The loops over the columns are unrolled as measured: aligned rows twice for 1, 4
// (TOP) and 8 queries (100000 x 768 bf16, 1 query: 70 -> 60 us, f32, 4 queries, TOP:
// 130 -> 120; not 300000 x 96 f32, 4 queries without TOP: 58 would be 67, nor
// 100000 x 768 f32, 1 query without TOP: 85 and 99), unaligned ones four times in 16
// bits (200000 x 75, 1 query: 38 -> 28; f32 with 8 queries would go from 66 to 85).
template <typename T, int NQ, bool VEC, bool TOP>
__global__ void __launch_bounds__(64)
    few_kernel(const T* __restrict__ x, size_t ld, int n, int d, const T* __restrict__ q,
               size_t ldq, int nq, float rf, const uint32_t* __restrict__ allowed,
               size_t ld_allowed, float4* __restrict__ part, float2* __restrict__ top,
               size_t groups, float* __restrict__ size, int* __restrict__ err) {
    wait_for_last();
    if (blockIdx.x == 0 && threadIdx.x == 0) *err = 0;  // (this path has no waits)
    constexpr int V = 16 / (int)sizeof(T);
    constexpr int RB = 8;
    constexpr bool PAIRS = NQ < 8;  // (two sums for each would not fit the registers)
    extern __shared__ float4 qs4[];
    float* qs = reinterpret_cast<float*>(qs4);  // [NQ][dp]
    const int dp = (d + 127) & ~127;
    for (int i = threadIdx.x; i < NQ * dp; i += 64) {
        const int j = i / dp, c = i - j * dp;
        qs[i] = j < nq && c < d ? to_f32<T>(q[(size_t)j * ldq + c]) : 0.0f;
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row_of_lane = ((lane >> 4 & 1) << 2 | (lane >> 3 & 1) << 1 | (lane >> 2 & 1)) +
                            8 * (lane & 3);
    Run r[NQ];
    float top_max[NQ];
    Largest<T> largest;  // of the rows that some query sees
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < NQ; ++j) r[j] = run_empty(), top_max[j] = NONE;
    const int ng = (n + GROUP - 1) / GROUP;
    for (int grp = blockIdx.x * 2 + warp; grp < ng; grp += gridDim.x * 2) {
        float sc[NQ];
#pragma unroll
        for (int j = 0; j < NQ; ++j) sc[j] = 0.0f;
        uint32_t seen = 0xffffffffu;
        if (TOP) {
            seen = 0u;
            for (int j = 0; j < (allowed && ld_allowed ? nq : 1); ++j)
                seen |= allowed_word(allowed, ld_allowed, j, (size_t)grp * GROUP, n);
        }
        const int first = TOP ? __ffs(seen) - 1 : 0;
#pragma unroll 1
        for (int b = 0; b < (seen ? 32 / RB : 0); ++b) {
            const int r0 = grp * GROUP + b * RB;
            uint64_t acc2[PAIRS ? NQ : 1][RB];  // sums of the even and of the odd columns
            float acc[NQ][RB];
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int i = 0; i < RB; ++i) {
                    acc[j][i] = 0.0f;
                    if (PAIRS) acc2[j][i] = 0ull;
                }
            const T* row[RB];
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                // (TOP: a row that no query sees is one that is seen, read again)
                const int at = TOP ? grp * GROUP + (seen >> (b * RB + i) & 1u ? b * RB + i : first)
                                   : min(r0 + i, n - 1);
                row[i] = x + (size_t)at * ld;
            }
            if (VEC) {
#pragma unroll ((NQ == 1 && (TOP || sizeof(T) == 2)) || (NQ == 4 && TOP) || NQ == 8 ? 2 : 1)
                for (int c = lane * V; c < d; c += 32 * V) {
                    uint4 xv[RB];
#pragma unroll
                    for (int i = 0; i < RB; ++i)
                        xv[i] = __ldg(reinterpret_cast<const uint4*>(row[i] + c));
                    if (TOP) {
#pragma unroll
                        for (int i = 0; i < RB; ++i) largest.add(xv[i]);
                    }
#pragma unroll
                    for (int h = 0; h < V; h += 4) {  // four columns at a time
                        uint64_t x01[RB], x23[RB];
#pragma unroll
                        for (int i = 0; i < RB; ++i) {
                            const T* e = reinterpret_cast<const T*>(&xv[i]) + h;
                            x01[i] = packf(to_f32<T>(e[0]), to_f32<T>(e[1]));
                            x23[i] = packf(to_f32<T>(e[2]), to_f32<T>(e[3]));
                        }
#pragma unroll
                        for (int j = 0; j < NQ; ++j) {
                            const float4 qv =
                                *reinterpret_cast<const float4*>(qs + j * dp + c + h);
                            const uint64_t q01 = packf(qv.x, qv.y), q23 = packf(qv.z, qv.w);
#pragma unroll
                            for (int i = 0; i < RB; ++i) {
                                if (PAIRS) {
                                    acc2[j][i] = fma2(x01[i], q01, acc2[j][i]);
                                    acc2[j][i] = fma2(x23[i], q23, acc2[j][i]);
                                } else {
                                    float a = acc[j][i];
                                    a = __fmaf_rn(lo_of(x01[i]), qv.x, a);
                                    a = __fmaf_rn(hi_of(x01[i]), qv.y, a);
                                    a = __fmaf_rn(lo_of(x23[i]), qv.z, a);
                                    acc[j][i] = __fmaf_rn(hi_of(x23[i]), qv.w, a);
                                }
                            }
                        }
                    }
                }
            } else {
#pragma unroll (sizeof(T) == 2 ? 4 : 1)
                for (int c = lane; c < d; c += 64) {  // columns c and c + 32
                    const bool two = c + 32 < d;
                    uint64_t xv[RB];
#pragma unroll
                    for (int i = 0; i < RB; ++i) {
                        const float x0 = to_f32<T>(row[i][c]);
                        const float x1 = two ? to_f32<T>(row[i][c + 32]) : 0.0f;
                        xv[i] = packf(x0, x1);
                        if (TOP) most = max3(most, fabsf(x0), fabsf(x1));
                    }
#pragma unroll
                    for (int j = 0; j < NQ; ++j) {
                        const float* qj = qs + j * dp + c;
                        const float qa = qj[0], qb = two ? qj[32] : 0.0f;
#pragma unroll
                        for (int i = 0; i < RB; ++i) {
                            if (PAIRS) acc2[j][i] = fma2(xv[i], packf(qa, qb), acc2[j][i]);
                            else
                                acc[j][i] = __fmaf_rn(hi_of(xv[i]), qb,
                                                      __fmaf_rn(lo_of(xv[i]), qa, acc[j][i]));
                        }
                    }
                }
            }
            if (PAIRS) {
#pragma unroll
                for (int j = 0; j < NQ; ++j)
#pragma unroll
                    for (int i = 0; i < RB; ++i) acc[j][i] = lo_of(acc2[j][i]) + hi_of(acc2[j][i]);
            }
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
                // halves of the rows are exchanged while more than one is left
                float t[RB];
#pragma unroll
                for (int i = 0; i < RB; ++i) t[i] = acc[j][i];
#pragma unroll
                for (int o = 16, m = RB / 2; o; o >>= 1, m >>= 1) {
                    if (m > 0) {
#pragma unroll
                        for (int i = 0; i < m; ++i) {
                            const float keep = lane & o ? t[i + m] : t[i];
                            const float give = lane & o ? t[i] : t[i + m];
                            t[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                        }
                    } else {
                        t[0] += __shfl_xor_sync(0xffffffffu, t[0], o);
                    }
                }
                if ((lane & (32 / RB - 1)) == b) sc[j] = t[0];
            }
        }
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            if (j >= nq) break;
            const uint32_t w =
                allowed_word(allowed, ld_allowed, j, (size_t)grp * GROUP, n);
            const bool ok = w >> row_of_lane & 1u;
            if (ok) {
                float dd = __fmaf_rn(sc[j], rf, -r[j].m);
                dd -= run_raise(r[j], dd);
                const float e = ex2(dd);
                r[j].l += e;
                r[j].a = __fmaf_rn(e, dd, r[j].a);
            }
            if (TOP) {
                float a = ok ? sc[j] * rf : NONE, b2 = NONE;
                a = __uint_as_float((__float_as_uint(a) & ~15u) | (unsigned)(row_of_lane >> 1));
#pragma unroll
                for (int o = 16; o; o >>= 1) {
                    const float oa = __shfl_xor_sync(0xffffffffu, a, o);
                    const float ob = __shfl_xor_sync(0xffffffffu, b2, o);
                    b2 = max3(b2, ob, fminf(a, oa));
                    a = fmaxf(a, oa);
                }
                if (lane == 0) top[(size_t)j * groups + grp] = make_float2(a, b2);
                if (a > NONE_BELOW) top_max[j] = fmaxf(top_max[j], unmarked(a));
            }
        }
    }
    // the lanes' triples joined, then the two warps'
    __shared__ Run other[NQ];
    __shared__ float other_top[NQ];
    __shared__ int other_size;
    const int size_all =
        __reduce_max_sync(0xffffffffu, __float_as_int(fmaxf(most, largest.get())));
    if (warp == 1 && lane == 0) other_size = size_all;
#pragma unroll
    for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            Run t;
            t.limit = __shfl_xor_sync(0xffffffffu, r[j].limit, o);
            t.m = __shfl_xor_sync(0xffffffffu, r[j].m, o);
            t.l = __shfl_xor_sync(0xffffffffu, r[j].l, o);
            t.a = __shfl_xor_sync(0xffffffffu, r[j].a, o);
            run_join(r[j], t);
        }
    if (warp == 1 && lane == 0)
#pragma unroll
        for (int j = 0; j < NQ; ++j) other[j] = r[j], other_top[j] = top_max[j];
    __syncthreads();
    if (warp == 0 && lane == 0)
#pragma unroll
        for (int j = 0; j < NQ; ++j)
            if (j < nq) {
                run_join(r[j], other[j]);
                part[(size_t)blockIdx.x * nq + j] =
                    run_stored(r[j], fmaxf(top_max[j], other_top[j]));
            }
    if (TOP && threadIdx.x == 0) size[blockIdx.x] = __int_as_float(max(size_all, other_size));
}

// ---------------------------------------------------------------------------
// joining the parts, the given row, the top alternatives
// ---------------------------------------------------------------------------
struct FinishArgs {
    const void *q, *x;
    size_t ldq, ldx;
    int q0, nq, n, d, k;
    float scale;
    const int64_t* targets;
    const uint32_t* allowed;
    size_t ld_allowed;
    const float4* part;
    int parts;
    const float* qf;
    const float2* top;
    size_t groups;
    // [sizes] whose largest bounds the elements of the rows that a query sees, null:
    // unknown.  Few queries: of the rows that one of them sees.  f32 rows on the
    // tensor cores: the rows' factors xf; with filters of their own those of all
    // rows, and a query that this sends to all groups takes its own.
    const float *size, *xf;
    int sizes;
    // Which groups a part folded.  Tensor-core pass: part i is quarter i % 4 of
    // the column tiles of chunk i / 4; few queries (nt = 0): part i is block i,
    // whose two warps took every 2 * parts-th group.
    int nt, chunks, per_tile, per_part;  // per_tile: groups of a tile, per_part: of its quarter
    double whole;  // a score over what its tensor-core sum comes to (see cut_of)
    float *logprob, *lse, *entropy, *top_logprob;
    int64_t* top_ids;
    const int* err;
};

// Order-preserving 32-bit image of a float.
__device__ __forceinline__ uint32_t ordered(float f) {
    const uint32_t u = __float_as_uint(f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
constexpr int PARTS_PICKED = 512;        // parts looked through at most
constexpr int PICKED = 256;              // groups picked for exact scoring at most
constexpr int CAND = 1024;               // rows scored exactly at once
constexpr int KEPT = 256;                // ... and ranked, as a rule

// Order-preserving 64-bit image of a double, and back: integer comparisons are
// what the ranking consists of.
__device__ __forceinline__ uint64_t ordered64(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double unordered64(uint64_t u) {
    return __longlong_as_double((long long)(u >> 63 ? u & 0x7fffffffffffffffull : ~u));
}

// q . x of ROWS rows in 64 bits (see Exact) over `lanes` lanes (a power of two).
// z: the largest element.
template <int ROWS, typename T>
__device__ __forceinline__ void dot_lanes(const T* const (&x)[ROWS],
                                          const typename Exact<T>::Q* q, int d, int sub, int lanes,
                                          bool wide, double (&s)[ROWS], Largest<T>& z) {
    constexpr int V = 16 / (int)sizeof(T);
    Exact<T> acc[ROWS][2];
    if (wide) {
        int c = sub * V;
        for (; c + V <= d; c += lanes * V) {
            uint4 raw[ROWS];
#pragma unroll
            for (int r = 0; r < ROWS; ++r) raw[r] = __ldg(reinterpret_cast<const uint4*>(x[r] + c));
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const T* e = reinterpret_cast<const T*>(&raw[r]);
#pragma unroll
                for (int i = 0; i < V; ++i) acc[r][i & 1].add(to_f32<T>(e[i]), q[c + i]);
                z.add(raw[r]);
            }
        }
        for (; c < d; ++c) {  // (the row's last, partial vector: one lane's)
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                acc[r][0].add(to_f32<T>(x[r][c]), q[c]);
                z.add(x[r][c]);
            }
        }
    } else {
#pragma unroll 4
        for (int c = sub; c < d; c += lanes)
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                acc[r][0].add(to_f32<T>(x[r][c]), q[c]);
                z.add(x[r][c]);
            }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        s[r] = acc[r][0].sum() + acc[r][1].sum();
        for (int o = lanes >> 1; o; o >>= 1) s[r] += __shfl_xor_sync(0xffffffffu, s[r], o);
    }
}

// One block per query: the partial triples joined, the groups that may hold
// one of the best k picked, their rows scored exactly and ranked.
//
// Picking needs no sort: the (k + PAD)th largest of 128 maxima over the parts
// is a bound that at least k + PAD groups reach, and for scores in no particular
// order hardly more do; only the groups of the parts that reach it are read.
//
// Bound by its chain of short dependent steps, half of whose time instructions
// are issued: 13 us for one query of 10000 x 128, 99 for 2048 of 131072 x 768
// (k = 20: some 60 rows a query gathered, 190 MB), 129 for 4096 of 262144 x 96.
// Seven blocks of 128 threads a multiprocessor (six: 126 and 145 us; eight spill:
// 110 and 170), one of 512 where there are fewer queries than that holds.
template <typename T, int THREADS_>
__global__ void __launch_bounds__(THREADS_, THREADS_ == 128 ? 7 : 1) finish_kernel(const FinishArgs p) {
    constexpr int W = THREADS_ / 32;
    extern __shared__ double qs_raw[];
    typename Exact<T>::Q* qs = reinterpret_cast<typename Exact<T>::Q*>(qs_raw);  // [dim]
    __shared__ __align__(16) float part_max[128];
    __shared__ float2 red[W];
    __shared__ float redf[W];
    __shared__ float s_bound;
    __shared__ int s_picked, s_cnt, s_parts;
    __shared__ int2 part_of[PARTS_PICKED];  // first group, groups
    __shared__ int sel[PICKED];
    __shared__ float2 sel_m[PICKED];
    __shared__ uint64_t cs[CAND + 1];  // exact scores, as ordered64
    __shared__ uint32_t ci[CAND + 1];
    __shared__ double s_kth;
    __shared__ int s_size;        // bits of the candidates' largest element
    __shared__ float s_qsize[W];  // parts of |q|^2
    __shared__ uint64_t kept[KEPT];
    __shared__ uint32_t kept_id[KEPT];
    __shared__ uint64_t set_max[128];
    __shared__ uint64_t s_least;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ql = blockIdx.x, q = p.q0 + ql;
    const T* qp = static_cast<const T*>(p.q) + (size_t)q * p.ldq;
    const T* xp = static_cast<const T*>(p.x);
    const uint32_t* al = p.allowed ? p.allowed + (size_t)q * p.ld_allowed : nullptr;
    const float2* top = p.k > 0 ? p.top + (size_t)ql * p.groups : nullptr;
    const int groups = p.k > 0 ? (int)p.groups : 0;
    float f = 1.0f;
    if (p.qf) f = p.qf[ql] == 0.0f ? 1.0f : p.qf[ql];
    const float rf = f * (float)((double)p.scale * LOG2E);
    // t was formed with rf, rounded to f32, from a sum that was cut; M of it is
    // set right here (t - M is small where it counts)
    const double unit = (double)p.scale * LOG2E;
    const double fix = (double)f * unit / (double)rf * p.whole;
    const int64_t target = p.targets ? p.targets[q] : -1;
    const bool given = target >= 0 && target < p.n;
    if (tid == 0) s_picked = s_cnt = s_parts = 0, s_kth = -INFINITY;
    float qq = 0.0f;
    for (int c = tid; c < p.d; c += THREADS_) {
        const float v = to_f32<T>(qp[c]);
        qs[c] = v;
        qq = __fmaf_rn(v, v, qq);
    }

    // ---- the largest reference, and the largest scores of 128 sets of parts ----
    float M = -INFINITY, gm = NONE;
    for (int i = tid; i < p.parts; i += THREADS_)
        M = fmaxf(M, p.part[(size_t)i * p.nq + ql].x);
    // (sets of parts where there are enough, else of groups)
    const bool by_parts = p.parts >= 128;
    if (tid < 128 && p.k > 0) {
        if (by_parts)
            for (int i = tid; i < p.parts; i += 128)
                gm = fmaxf(gm, p.part[(size_t)i * p.nq + ql].w);
        else
#pragma unroll 4
            for (int i = tid; i < groups; i += 128) gm = fmaxf(gm, unmarked(top[i].x));
        part_max[tid] = gm;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
#pragma unroll
    for (int o = 16; o; o >>= 1) qq += __shfl_xor_sync(0xffffffffu, qq, o);
    if (lane == 0) redf[warp] = M, s_qsize[warp] = qq;
    if (tid == 0) s_size = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) M = fmaxf(M, redf[i]);
    // ---- the sums over the parts, in units of 2^M ----
    float L = 0.0f, A = 0.0f;
    if (p.size) {
        float z = 0.0f;
        for (int i = tid; i < p.sizes; i += THREADS_) {
            const float v = p.size[i];  // (infinite: of a row that makes its queries NaN)
            if (v <= FLT_MAX) z = fmaxf(z, v);
        }
        const int w = __reduce_max_sync(0xffffffffu, __float_as_int(z));
        if (lane == 0) atomicMax(&s_size, w);
    }
    for (int i = tid; i < p.parts; i += THREADS_) {
        const float4 t = p.part[(size_t)i * p.nq + ql];
        if (t.y == 0.0f && t.z == 0.0f) continue;
        const float d = t.x == M ? 0.0f : t.x - M, e = ex2(d);
        L = __fmaf_rn(t.y, e, L);
        A = __fmaf_rn(__fmaf_rn(d, t.y, t.z), e, A);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        L += __shfl_xor_sync(0xffffffffu, L, o);
        A += __shfl_xor_sync(0xffffffffu, A, o);
    }
    if (lane == 0) red[warp] = make_float2(L, A);
    if (p.k > 0 && tid < 128) {
        // (equal ones all write the same)
        int above = 0, from = 0;
        const float mine = part_max[tid];
        const float4* all = reinterpret_cast<const float4*>(part_max);
#pragma unroll 8
        for (int i = 0; i < 32; ++i) {
            const float4 v = all[i];
            above += (v.x > mine) + (v.y > mine) + (v.z > mine) + (v.w > mine);
            from += (v.x >= mine) + (v.y >= mine) + (v.z >= mine) + (v.w >= mine);
        }
        if (above < p.k + PAD && p.k + PAD <= from) s_bound = mine;
    }
    __syncthreads();
    L = A = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) L += red[i].x, A += red[i].y;
    const bool none = L == 0.0f;  // no row may be seen
    const bool bad = !(A == A) || !(L == L) || (p.err && *p.err != 0);
    // log2 of L by its exponent and its fraction: the large part is exact
    double lg = 0.0;
    if (!none && !bad) {
        const int e = ilogbf(L);
        lg = (double)e + (double)log2f(ldexpf(L, -e));
    }
    const double lse = bad ? NAN : none ? -INFINITY : LN2 * ((double)M * fix + lg);
    if (tid == 0) {
        if (p.lse) p.lse[q] = (float)lse;
        if (p.entropy) p.entropy[q] = (float)(bad ? NAN : none ? 0.0 : LN2 * (lg - (double)(A / L)));
    }

    // rows ci[from, to) scored exactly
    const bool wide = ((reinterpret_cast<uintptr_t>(xp) | (p.ldx * sizeof(T))) & 15) == 0;
    const int lanes = p.d * (int)sizeof(T) <= 512 ? 8 : 32;
    const int sub = lane & (lanes - 1);
    auto score = [&](int from, int to) {
        constexpr int ROWS = 4;
        Largest<T> largest;
        const int per = THREADS_ / lanes;
        for (int i = from; i < to; i += ROWS * per) {
            const T* x[ROWS];
            double v[ROWS];
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const int j = i + r * per + tid / lanes;
                x[r] = xp + (size_t)ci[j < to ? j : from] * p.ldx;
            }
            dot_lanes<ROWS, T>(x, qs, p.d, sub, lanes, wide, v, largest);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const int j = i + r * per + tid / lanes;
                if (sub == 0 && j < to) cs[j] = ordered64(v[r]);
            }
        }
        if (p.k > 0 && !p.xf) {
            const int w = __reduce_max_sync(0xffffffffu, __float_as_int(largest.get()));
            if (lane == 0) atomicMax(&s_size, w);
        }
    };
    auto seen = [&](uint32_t id) {
        return id < (uint32_t)p.n && (!al || (al[id >> 5] >> (id & 31) & 1u));
    };

    // ---- groups that reach the bound, the marked pair of each a candidate ----
    const float bound = p.k > 0 && !bad ? s_bound : INFINITY;
    auto pick = [&](int gi, float2 m) {
        if (m.x > NONE_BELOW && unmarked(m.x) >= bound) {
            const int at = atomicAdd(&s_picked, 1);
            if (at < PICKED) sel[at] = gi, sel_m[at] = m;
        }
    };
    if (!by_parts) {
#pragma unroll 4
        for (int i = tid; i < groups; i += THREADS_) pick(i, top[i]);
    }
    // a part's groups are `run` side by side, `step` from one run to the next
    const int run = p.nt ? p.per_part : 2, step = p.nt ? p.per_tile : 2 * p.parts;
    for (int i = tid; i < (groups && by_parts ? p.parts : 0); i += THREADS_) {
        const float t = p.part[(size_t)i * p.nq + ql].w;
        if (t > NONE_BELOW && t >= bound) {
            const int at = atomicAdd(&s_parts, 1);
            if (at >= PARTS_PICKED) continue;
            if (p.nt) {
                const long long c = i >> 2;
                const int t0 = (int)(c * p.nt / p.chunks), t1 = (int)((c + 1) * p.nt / p.chunks);
                part_of[at] = make_int2(t0 * step + (i & 3) * run, (t1 - t0) * run);
            } else {
                part_of[at] = make_int2(2 * i, 2 * ((groups + step - 1) / step));
            }
        }
    }
    __syncthreads();
    const int nparts = min(s_parts, PARTS_PICKED), few = run >> 1;  // (run: 1 or 2)
    for (int i = tid >> 4; i < nparts; i += THREADS_ / 16) {
        const int2 part = part_of[i];
#pragma unroll 4
        for (int e = tid & 15; e < part.y; e += 16) {
            const int gi = part.x + (e >> few) * step + (e & few);
            if (gi < groups) pick(gi, __ldg(top + gi));
        }
    }
    __syncthreads();
    const int picked = s_picked;
    bool all_groups = picked > PICKED || s_parts > PARTS_PICKED;  // (many equal scores)
    if (!all_groups && tid < picked) {
        const uint32_t pair = __float_as_uint(sel_m[tid].x) & 15u;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t id = (uint32_t)sel[tid] * GROUP + pair * 2 + h;
            if (seen(id)) ci[atomicAdd(&s_cnt, 1)] = id;
        }
    }
    if (THREADS_ < PICKED && !all_groups && tid + THREADS_ < picked) {
        const uint32_t pair = __float_as_uint(sel_m[tid + THREADS_].x) & 15u;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t id = (uint32_t)sel[tid + THREADS_] * GROUP + pair * 2 + h;
            if (seen(id)) ci[atomicAdd(&s_cnt, 1)] = id;
        }
    }
    __syncthreads();
    // the row whose log probability is asked for comes last (a row that the query
    // may not see is not looked at: what it holds would count as a candidate's size)
    const int cnt = s_cnt;
    const bool last = given && seen((uint32_t)target);
    if (tid == 0 && last) ci[cnt] = (uint32_t)target;
    __syncthreads();
    if (cnt + last > 0) score(0, cnt + last);
    __syncthreads();
    if (tid == 0 && p.logprob) {
        float v = bad ? NAN : 0.0f;
        if (given && !bad)
            v = last ? (float)(unordered64(cs[cnt]) * (double)p.scale - lse) : -INFINITY;
        p.logprob[q] = v;
    }
    if (p.k == 0) return;

    // give(i, rank of candidate i among the first n), eight lanes a candidate
    auto rank_all = [&](int n, auto&& give) {
        for (int i0 = 0; i0 < n; i0 += THREADS_ / 8) {
            const int i = i0 + tid / 8, at = min(i, n - 1);
            const uint64_t v = cs[at];
            const uint32_t id = ci[at];
            int rank = 0;
            for (int j = tid & 7; j < n; j += 8) {
                const uint64_t o = cs[j];
                rank += o > v || (o == v && ci[j] < id);
            }
            rank += __shfl_xor_sync(0xffffffffu, rank, 1);
            rank += __shfl_xor_sync(0xffffffffu, rank, 2);
            rank += __shfl_xor_sync(0xffffffffu, rank, 4);
            if (i < n && (tid & 7) == 0) give(i, rank);
        }
    };
    // Of the first n candidates those of at least `least` (at least k), moved to
    // the front if they are at most KEPT: ranking costs their number squared.
    // Returns how many are left.
    auto narrow = [&](int n, uint64_t least) -> int {
        __syncthreads();
        if (tid == 0) s_parts = 0;
        __syncthreads();
        for (int i = tid; i < n; i += THREADS_)
            if (cs[i] >= least) {
                const int at = atomicAdd(&s_parts, 1);
                if (at < KEPT) kept[at] = cs[i], kept_id[at] = ci[i];
            }
        __syncthreads();
        const int left = s_parts;
        if (left > KEPT) return n;
        for (int i = tid; i < left; i += THREADS_) cs[i] = kept[i], ci[i] = kept_id[i];
        __syncthreads();
        return left;
    };
    // The kth largest of 128 maxima over interleaved sets of n > 128 candidates:
    // at least k reach it.
    auto least_of = [&](int n) -> uint64_t {
        if (tid < 128) {
            uint64_t m = 0;
            for (int i = tid; i < n; i += 128) m = max(m, cs[i]);
            set_max[tid] = m;
        }
        __syncthreads();
        if (tid < 128) {
            const uint64_t m = set_max[tid];
            int rank = 0;
#pragma unroll 8
            for (int i = 0; i < 128; ++i)
                rank += set_max[i] > m || (set_max[i] == m && i < tid);
            if (rank == p.k - 1) s_least = m;
        }
        __syncthreads();
        return s_least;
    };
    // Whether a score of at most `m` (as a group left it) may be among the best
    // k, whose last exact score so far is s_kth: a mark moves it by 2^-19 of
    // itself, the 32-bit sums by less than 2^-18 of |q| sqrt(d) max |x_c|, x the
    // rows that the query sees.  The tensor cores read 16-bit rows as they are,
    // so nothing has looked at their sizes: x then are those scored so far, and a
    // row whose elements are many times theirs may be passed over if its score is
    // above the kth by less than its own error.  (A pass for the sizes alone
    // would read the rows again: 100003 x 768 with 8 queries 55 us and 24 more.)
    qq = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) qq += s_qsize[i];
    auto may_enter = [&](double m) {
        const double v = m / unit, kth = s_kth;
        const double size = (double)sqrtf(qq * (float)p.d) * (double)__int_as_float(s_size) *
                            (p.xf ? 16384.0 : 1.0);  // (packed: below 2^14 of the factor)
        return !(v < kth - (fabs(v) + fabs(kth)) * 0x1p-16 - size * 0x1p-18);
    };
    const int ranked = cnt > 128 ? narrow(cnt, least_of(cnt)) : cnt;
    const int best = min(ranked, p.k);
    rank_all(ranked, [&](int i, int rank) {
        if (rank < p.k) kept[rank] = cs[i], kept_id[rank] = ci[i];
        if (rank == p.k - 1) s_kth = unordered64(cs[i]);
    });
    if (tid == 0) s_parts = best;
    __syncthreads();
    // ---- groups whose second largest score may still enter: their other rows ----
    bool more = bound > NONE_BELOW && may_enter(bound);  // groups below the bound may
    if ((more || all_groups) && !bad && p.xf && p.ld_allowed) {
        __syncthreads();
        if (tid == 0) s_size = 0;
        __syncthreads();
        float z = 0.0f;
        for (int j = tid; j < p.n; j += THREADS_)
            if (al[j >> 5] >> (j & 31) & 1u) z = fmaxf(z, p.xf[j]);
        const int w = __reduce_max_sync(0xffffffffu, __float_as_int(z));
        if (lane == 0) atomicMax(&s_size, w);
        __syncthreads();
        more = bound > NONE_BELOW && may_enter(bound);
    }
    if (!all_groups && !more && !bad) {
        for (int i = tid; i < picked; i += THREADS_) {
            const float2 m = sel_m[i];
            if (!(m.y > NONE_BELOW) || !may_enter(m.y)) continue;
            const uint32_t pair = __float_as_uint(m.x) & 15u, g0 = (uint32_t)sel[i] * GROUP;
            uint32_t rest = allowed_word(al, 0, 0, g0, p.n) & ~(3u << (2 * pair));
            int at = atomicAdd(&s_cnt, __popc(rest));
            while (rest) {
                if (at < CAND) ci[at] = g0 + (uint32_t)(__ffs(rest) - 1);
                ++at;
                rest &= rest - 1;
            }
        }
        __syncthreads();
        if (s_cnt <= CAND) {
            score(cnt, s_cnt);
            __syncthreads();
            // those that do, behind the best so far
            const uint64_t least = best == p.k ? kept[p.k - 1] : 0;
            for (int i = cnt + tid; i < s_cnt; i += THREADS_) {
                if (cs[i] < least) continue;
                const int at = atomicAdd(&s_parts, 1);
                if (at < KEPT) kept[at] = cs[i], kept_id[at] = ci[i];
            }
        }
    }
    __syncthreads();
    const int total = s_parts;
    all_groups = !bad && (all_groups || more || s_cnt > CAND || total > KEPT);
    __syncthreads();
    if (all_groups) {
        // ---- too many groups are as good (many equal or nearly equal scores, or
        // hardly more groups than k): every row of every group that may enter is
        // scored, as many at a time as there is room for, the best k kept ----
        if (tid == 0) s_cnt = 0;
        __syncthreads();
        const int step = (CAND - FDB_MAX_ALTERNATIVES) / GROUP;
        for (int g0 = 0; g0 < groups; g0 += step) {
            const int kept_now = s_cnt;
            __syncthreads();
            for (int gi = g0 + warp; gi < min(groups, g0 + step); gi += W) {
                const float m1 = top[gi].x;
                if (!(m1 > NONE_BELOW) || !may_enter(m1)) continue;
                const uint32_t w = allowed_word(al, 0, 0, (size_t)gi * GROUP, p.n);
                int at = 0;
                if (lane == 0) at = atomicAdd(&s_cnt, __popc(w));
                at = __shfl_sync(0xffffffffu, at, 0) + __popc(w & ((1u << lane) - 1u));
                if (w >> lane & 1u) ci[at] = (uint32_t)gi * GROUP + (uint32_t)lane;
            }
            __syncthreads();
            const int have = s_cnt;
            if (have == kept_now) continue;  // (the same for all threads)
            score(kept_now, have);
            __syncthreads();
            int left = have;
            if (have > KEPT) left = narrow(have, least_of(have));
            rank_all(left, [&](int i, int rank) {
                if (rank < p.k) kept[rank] = cs[i], kept_id[rank] = ci[i];
            });
            __syncthreads();
            const int keep = min(left, p.k);
            for (int i = tid; i < keep; i += THREADS_) cs[i] = kept[i], ci[i] = kept_id[i];
            if (tid == 0) {
                s_cnt = keep;
                if (keep == p.k) s_kth = unordered64(kept[p.k - 1]);
            }
            __syncthreads();
        }
        __syncthreads();
    }
    // ---- written in order ----
    const int have = bad ? 0 : all_groups ? s_cnt : total;
    auto write = [&](int rank, uint64_t score, uint32_t id) {
        if (rank >= p.k) return;
        p.top_ids[(size_t)q * p.k + rank] = (int64_t)id;
        p.top_logprob[(size_t)q * p.k + rank] =
            (float)(unordered64(score) * (double)p.scale - lse);
    };
    if (all_groups) {  // (at most k, ranked in the last round)
        for (int i = tid; i < have; i += THREADS_) write(i, cs[i], ci[i]);
    } else if (total == best) {
        for (int i = tid; i < have; i += THREADS_) write(i, kept[i], kept_id[i]);
    } else {
        for (int i = tid; i < have; i += THREADS_) cs[i] = kept[i], ci[i] = kept_id[i];
        __syncthreads();
        rank_all(have, [&](int i, int rank) { write(rank, cs[i], ci[i]); });
    }
    for (int i = have + tid; i < p.k; i += THREADS_) {
        p.top_ids[(size_t)q * p.k + i] = -1;
        p.top_logprob[(size_t)q * p.k + i] = bad ? NAN : -INFINITY;
    }
}

// ---------------------------------------------------------------------------
// backward: what the products need
// ---------------------------------------------------------------------------
// Rows some query may see: the OR of the filters, 32 words a block, 32 queries
// at a time (latency-bound: 777 filters of 20003 rows took 15.4 us eight at a
// time, 4.6 now).
__global__ void __launch_bounds__(1024)
    any_kernel(const uint32_t* __restrict__ allowed, size_t ld, int nq, size_t words,
               uint32_t* __restrict__ out) {
    __shared__ uint32_t part[32][33];
    const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
    const size_t w = (size_t)blockIdx.x * 32 + lane;
    uint32_t r = 0;
    if (w < words) {
#pragma unroll 8
        for (int q = row; q < nq; q += 32) r |= __ldg(allowed + (size_t)q * ld + w);
    }
    part[row][lane] = r;
    __syncthreads();
    r = __reduce_or_sync(0xffffffffu, part[lane][row]);
    const size_t o = (size_t)blockIdx.x * 32 + row;
    if (lane == 0 && o < words) out[o] = r;
    wait_for_last();  // (beside the kernel before it)
}
struct CoefArgs {
    int nq, n;
    double scale, whole;  // (whole: see cut_of)
    const float *lse, *entropy, *d_logprob, *d_lse, *d_entropy;
    const int64_t* targets;
    const uint32_t* allowed;
    size_t ld_allowed;
    Coef* out;
    float* rest;  // nullable
    const float* at_least;  // nullable, see GivenRows
};
// What reaches a query's scores, and a bound B of its G's size (p |lp| <= 1/e).
struct Upstream {
    double dl, g, dh, H;
    int target;
    bool empty;
    float bound;
};
__device__ __forceinline__ Upstream upstream_of(const CoefArgs& a, int i) {
    // (all loads but the filter's first: one after the other they take 2 us more)
    const float lse = a.lse[i];
    const int64_t t = a.targets ? a.targets[i] : -1;
    const float g = a.d_logprob ? a.d_logprob[i] : 0.0f, dl = a.d_lse ? a.d_lse[i] : 0.0f;
    const float dh = a.d_entropy ? a.d_entropy[i] : 0.0f;
    const float H = a.d_entropy ? a.entropy[i] : 0.0f;
    Upstream u;
    u.empty = lse == -INFINITY;
    const bool given = !u.empty && t >= 0 && t < a.n &&
                       (!a.allowed ||
                        (a.allowed[(size_t)i * a.ld_allowed + (size_t)(t >> 5)] >> (t & 31) & 1u));
    u.g = given ? g : 0.0;
    u.dl = u.empty ? 0.0 : dl;
    u.dh = u.empty ? 0.0 : dh;
    u.H = u.dh != 0.0 ? (double)H : 0.0;
    u.target = given ? (int)t : -1;
    u.bound = (float)(a.scale * (fabs(u.dl) + 2.0 * fabs(u.g) + fabs(u.dh) * (fabs(u.H) + 1.0)));
    if (a.at_least) u.bound = fmaxf(u.bound, (float)(a.scale * (double)a.at_least[i]));
    return u;
}
// G_ij = scale [ p_ij (dl - g - h (lp_ij + H)) + g 1{j = t} ] with lp = ln2 x:
// = p (c + h' x) + g'; times w.  f: a score over its sum of packed products.
__device__ __forceinline__ Coef coef_of(const CoefArgs& a, int i, double f, double w) {
    const Upstream u = upstream_of(a, i);
    const float lse = a.lse[i];
    const double rf = f * a.scale * LOG2E * a.whole, l = (double)lse * LOG2E;
    Coef k;
    k.rf_hi = (float)rf;
    k.rf_lo = (float)(rf - (double)k.rf_hi);
    k.l_hi = u.empty ? INFINITY : (float)l;
    k.l_lo = u.empty ? 0.0f : (float)(l - (double)k.l_hi);
    k.c = lse == lse ? (float)(a.scale * w * (u.dl - u.g - u.dh * u.H)) : NAN;
    k.h = (float)(-a.scale * w * u.dh * LN2);
    k.g = (float)(a.scale * w * u.g);
    k.target = u.target;
    return k;
}
// Clears the head of the workspace, marks the queries that see anything, as bits
// (an empty one is taken as zeros, so that what it holds cannot set the scale of
// the others), and leaves the exponent of each query's B.
__global__ void head_kernel(const CoefArgs a, uint32_t* __restrict__ alive,
                            int* __restrict__ weight, uint32_t* __restrict__ head,
                            int head_words) {
    wait_for_last();
    const int q = blockIdx.x * blockDim.x + threadIdx.x;
    if (q < head_words) head[q] = 0u;
    bool on = false;
    if (q < a.nq) {
        const Upstream u = upstream_of(a, q);
        on = !u.empty;
        weight[q] = weight_of(u.bound);
    }
    const unsigned b = __ballot_sync(0xffffffffu, on);
    if ((threadIdx.x & 31) == 0 && q < a.nq) alive[q >> 5] = b;
}
// The scales of what is stored.  With rows x_j = 2^-ej xp_j and queries
// q_i = 2^-ei qp_i (packed), X the largest 2^-ej and f_j = 2^-ej / X:
//
//   G'_ij = G_ij f_j W_i,   W_i = 2^13 / B_i to a power of two
//   d_queries_i = X / W_i sum_j G'_ij xp_j
//   d_rows_j = M 2^-13 / f_j sum_i G'_ij qs_i,   qs_i = qp_i 2^-ei B_i / M
//
// M the largest 2^-ei B_i.  Every query's largest |G'| comes to [2^13, 2^15)
// whatever the others' upstream gradients are (with one factor for all, a query
// with 1e-6 of the largest had its d_queries off by 4e-3 of themselves in f32);
// d_rows' sums, over queries, hold the terms of each to fp16's least step in the
// scale of the largest, 2^-37 of it.
//
// A row far below the largest would leave too few bits in G'.  Such a row (below
// 2^-4 of the largest scale) takes a larger one and is shifted down instead;
// rows of zeros or with a NaN, whose elements are zeros, take any.  Almost none
// has work.  One warp per query: its copy qs, its coefficients; one per 32 rows.
__global__ void __launch_bounds__(256)
    settle_kernel(const CoefArgs a, const __half* __restrict__ qp, const float* __restrict__ qf,
                  const int* __restrict__ weight, __half* __restrict__ qs,
                  float* __restrict__ out_f, __half* __restrict__ xp, float* __restrict__ xf,
                  int kp, int parts, int qblocks, const GradHead* __restrict__ head) {
    wait_for_last();
    qp = here(qp), qf = here(qf), weight = here(weight), xp = here(xp), xf = here(xf);
    head = here(head);
    const int lane = threadIdx.x & 31;
    const float mx = head->x_most;
    const int lx = mx > 0.0f ? ilogbf(mx) : 0;
    if ((int)blockIdx.x < qblocks) {
        const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
        if (row >= a.nq) return;
        const float f = qf[row];
        const bool none = weight[row] == NO_WEIGHT;
        const int e = none ? 13 : weight[row];
        if (lane == 0) {
            a.out[row] = coef_of(a, row, ldexp((double)f, lx), ldexp(1.0, 13 - e));
            out_f[row] = ldexpf(1.0f, min(lx - 13 + e, 127));
            if (a.rest) a.rest[row] = 0.0f;
        }
        const float s = none || !(f > 0.0f)
                            ? 0.0f
                            : ldexpf(1.0f, ilogbf(f) + e + WEIGHT_ZERO - (int)head->q_most);
        const size_t at = (size_t)row * (size_t)(parts * kp);
        for (int c = lane * 8; c < kp; c += 256) {
            __align__(16) __half hi[8], lo[8];
            *reinterpret_cast<uint4*>(hi) = *reinterpret_cast<const uint4*>(qp + at + c);
            if (parts == 2)
                *reinterpret_cast<uint4*>(lo) = *reinterpret_cast<const uint4*>(qp + at + kp + c);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float v = __half2float(hi[i]) * s;
                if (parts == 2) v = __fmaf_rn(__half2float(lo[i]), s, v);
                hi[i] = __float2half_rn(v);
                lo[i] = __float2half_rn(v - __half2float(hi[i]));
            }
            *reinterpret_cast<uint4*>(qs + at + c) = *reinterpret_cast<const uint4*>(hi);
            if (parts == 2)
                *reinterpret_cast<uint4*>(qs + at + kp + c) = *reinterpret_cast<const uint4*>(lo);
        }
        return;
    }
    // rows: a lane looks at one, the warp shifts those that need it
    const int row0 = (((int)blockIdx.x - qblocks) * 8 + (threadIdx.x >> 5)) * 32;
    const int row = row0 + lane;
    const float least = mx * 0x1p-4f, v = row < a.n ? xf[row] : 0.0f;
    const bool small = v > 0.0f && v < least;
    unsigned todo = __ballot_sync(0xffffffffu, small);
    while (todo) {
        const int r = __ffs(todo) - 1, width = parts * kp;
        const float s = __shfl_sync(0xffffffffu, v, r) / least;
        __half* h = xp + (size_t)(row0 + r) * width;
        for (int c = lane; c < width; c += 32) h[c] = __float2half_rn(__half2float(h[c]) * s);
        todo &= todo - 1;
    }
    if (row < a.n) xf[row] = !(v > 0.0f) ? 1.0f : small ? 0x1p-4f : ldexpf(v, -lx);
}
// The score gradients at rows that are given with theirs (see GivenRows), one warp
// per query, over what GRAD has left there.  One part: the largest of what fp16
// leaves of a query's is added to its d_queries, as GRAD's given row's is (one of
// them is most of the sum where it counts).
struct GivenArgs {
    GivenRows given;
    int nq;
    const int* weight;
    const float* xf;  // (as settle_kernel left them)
    __half* gr;
    size_t ldg;
    int nqp, parts, j0, cols;  // this chunk
    float* rest;               // of all chunks, and its row; null: not now
    int* rest_row;
};
__global__ void __launch_bounds__(256) given_kernel(const GivenArgs p) {
    wait_for_last();
    const int lane = threadIdx.x & 31, q = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (q >= p.nq) return;
    const int e = p.weight[q];
    const float w = e == NO_WEIGHT ? 1.0f : ldexpf(1.0f, min(13 - e, 127));
    const size_t at = (size_t)q * p.given.k;
    float most = 0.0f;
    int most_row = -1;
    for (int i = lane; i < p.given.k; i += 32) {
        const int row = p.given.row[at + i];
        if (row < 0) continue;
        const float v = p.given.g[at + i] * w * p.xf[row];
        const __half hi = __float2half_rn(v);
        const float left = v - __half2float(hi);
        const int col = row - p.j0;
        if ((unsigned)col < (unsigned)p.cols) {
            p.gr[(size_t)q * p.ldg + col] = hi;
            if (p.parts == 2)
                p.gr[(size_t)(p.nqp + q) * p.ldg + col] = __float2half_rn(left);
        }
        if (fabsf(left) > fabsf(most)) most = left, most_row = row;
    }
    if (!p.rest) return;
    const float top = __int_as_float(__reduce_max_sync(0xffffffffu, __float_as_int(fabsf(most))));
    const unsigned who = __ballot_sync(0xffffffffu, most_row >= 0 && fabsf(most) == top);
    if (who && lane == __ffs(who) - 1) {
        p.rest[q] = most;
        p.rest_row[q] = most_row;
    }
}
// d_queries of 16-bit inputs: rest[r] times the given row is added (see GRAD).
struct JoinRest {
    const float* rest;  // null: nothing
    const int* row;     // `step` apart
    int step;
    const __half* x;
    int ldx;
};
// Sum of the splits, scaled (f null: not), in the output's type: four columns of a row by one
// thread, or by eight that take every eighth split and are added in order (16
// splits and more: 64 of 100 x 128 took 10.9 us one after the other, now 3.7;
// few splits of a large output are better off with more columns a block).
template <int TURNS>
__global__ void __launch_bounds__(256)
    join_kernel(const float* __restrict__ partial, int splits, int rows, int cols,
                const float* __restrict__ f, const GradHead* __restrict__ head, void* out,
                size_t ldo, int dtype, const JoinRest rest) {
    wait_for_last();
    partial = here(partial), f = here(f), head = here(head);
    constexpr int LANES = 256 / TURNS;
    __shared__ float4 part[TURNS][LANES];
    const unsigned per4 = (unsigned)(cols + 3) / 4;
    const size_t plane = (size_t)rows * cols, all = (size_t)rows * per4;
    const bool wide = (cols & 3) == 0;
    const int lane = threadIdx.x % LANES, turn = threadIdx.x / LANES;
    for (size_t i0 = (size_t)blockIdx.x * LANES; i0 < all; i0 += (size_t)gridDim.x * LANES) {
        const size_t i = i0 + lane;
        const size_t r = i / per4;
        const int k = (int)(i - r * per4) * 4;
        const float* src = partial + r * cols + k;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (i < all) {
            if (wide) {
#pragma unroll 4
                for (int j = turn; j < splits; j += TURNS) {
                    const float4 t = __ldcs(reinterpret_cast<const float4*>(src + j * plane));
                    v.x += t.x, v.y += t.y, v.z += t.z, v.w += t.w;
                }
            } else {
                for (int j = turn; j < splits; j += TURNS) {
                    const float* t = src + j * plane;
                    v.x += t[0];
                    if (k + 1 < cols) v.y += t[1];
                    if (k + 2 < cols) v.z += t[2];
                    if (k + 3 < cols) v.w += t[3];
                }
            }
        }
        if (TURNS > 1) {
            part[turn][lane] = v;
            __syncthreads();
        }
        if (turn == 0 && i < all) {
            for (int j = 1; j < TURNS; ++j) {
                const float4 t = part[j][lane];
                v.x += t.x, v.y += t.y, v.z += t.z, v.w += t.w;
            }
            if (rest.rest) {
                const float g = rest.rest[r];
                if (g != 0.0f) {
                    const __half* x = rest.x + (size_t)rest.row[r * rest.step] * rest.ldx + k;
                    v.x = __fmaf_rn(g, __half2float(x[0]), v.x);
                    if (k + 1 < cols) v.y = __fmaf_rn(g, __half2float(x[1]), v.y);
                    if (k + 2 < cols) v.z = __fmaf_rn(g, __half2float(x[2]), v.z);
                    if (k + 3 < cols) v.w = __fmaf_rn(g, __half2float(x[3]), v.w);
                }
            }
            const float s = f ? out_factor(f[r], head) : 1.0f;
            const float o[4] = {v.x * s, v.y * s, v.z * s, v.w * s};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (k + e < cols) put(out, r * ldo + k + e, dtype, o[e]);
        }
        if (TURNS > 1) __syncthreads();
    }
}
static void launch_join(cudaStream_t s, int sms, const float* partial, int splits, int rows,
                        int cols, const float* f, const GradHead* head, void* out, size_t ldo,
                        int dtype, const JoinRest& rest = JoinRest{}) {
    if (splits >= 16)
        launch(true, s, join_kernel<8>, sms * 8, 256, 0, partial, splits, rows, cols, f, head, out,
               ldo, dtype, rest);
    else
        launch(true, s, join_kernel<1>, sms * 8, 256, 0, partial, splits, rows, cols, f, head, out,
               ldo, dtype, rest);
}
// ---------------------------------------------------------------------------
// the gradient for a few queries: one pass over the rows on the FMA pipes
// ---------------------------------------------------------------------------
// A block takes 16 rows at a time.  Each warp forms the scores of two of them
// (its lanes share the columns) while it lays them into shared memory, and the
// score gradients; then a thread owns four columns of the 16 rows (or of a share
// of them, if the columns are few): d_rows = G^T Q is complete and stored, its
// columns of d_queries = G X stay in registers until the block's last rows.
// Every row is read and its gradient written once; what bounds it is the latency
// of the two halves, which the blocks of a multiprocessor (registers: three of 1
// or 2 queries, two of more) hide for each other: 100000 x 768 f32 takes 132 us
// with 1 query and 252 with 8, where the bytes alone take 92 (bf16: 113 and 250, 46).
// The tensor-core path copies the rows and pads the queries to 256: see FEW_GRAD.
template <typename T>
struct FewGrad {
    const T* x;
    size_t ldx;
    const T* q;
    size_t ldq;
    int n, d, nq;
    CoefArgs coef;
    T* dx;           // nullable
    size_t ld_dx;
    float* partial;  // [blocks][nq][d], nullable
    int* err;
    GivenRows given;
};
constexpr int FEW_ROWS = 16;
constexpr int few_per_sm(int NQ) { return NQ <= 2 ? 3 : 2; }  // (blocks; registers)
static size_t few_grad_smem(int NQ, size_t d, size_t elem) {
    const size_t dp = (d + 63) / 64 * 64;
    return NQ * dp * 4 + FEW_ROWS * NQ * 8 +
           std::max<size_t>(FEW_ROWS * dp * elem, (size_t)NQ * 4096);
}
// Columns c and c + 32 of a query lie side by side, as the lanes multiply two
// at a time.
__device__ __forceinline__ int few_at(int c) {
    return (c & ~63) + 2 * (c & 31) + (c >> 5 & 1);
}
// GIVEN: with score gradients at given rows.  Each thread looks after up to NQ of
// them (at most 256 a query) and lays those of the block's rows over the others.
template <typename T, int NQ, bool GIVEN>
__global__ void __launch_bounds__(256, few_per_sm(NQ)) few_grad_kernel(const FewGrad<T> p) {
    wait_for_last();
    extern __shared__ float4 few_raw[];
    const int d = p.d, ct_n = (d + 3) / 4, dp = (d + 63) & ~63;
    float* qs = reinterpret_cast<float*>(few_raw);                  // [NQ][dp], see few_at
    float2* gs = reinterpret_cast<float2*>(qs + NQ * dp);           // [rows][NQ], twice each
    T* xs = reinterpret_cast<T*>(gs + FEW_ROWS * NQ);               // [rows][dp], at the end sums
    __shared__ Coef co[NQ];
    __shared__ int q_bad[NQ], x_bad[FEW_ROWS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (blockIdx.x == 0 && tid == 0) *p.err = 0;  // (this path has no waits)
    if (tid < NQ) q_bad[tid] = 0;
    __syncthreads();
    for (int i = tid; i < NQ * dp; i += 256) {
        const int j = i / dp, c = i - j * dp;
        const float v = j < p.nq && c < d ? to_f32<T>(p.q[(size_t)j * p.ldq + c]) : 0.0f;
        if (!(fabsf(v) <= FLT_MAX)) q_bad[j] = 1;
        qs[j * dp + few_at(c)] = v;
    }
    if (tid < p.nq) {
        co[tid] = coef_of(p.coef, tid, 1.0, 1.0);
    }
    __syncthreads();
    // what a query that sees nothing holds does not count, an infinity or NaN of
    // another reaches the rows that it sees through G alone
    for (int i = tid; i < NQ * dp; i += 256) {
        const int j = i / dp;
        if (j < p.nq && (q_bad[j] || p.coef.lse[j] == -INFINITY)) qs[i] = 0.0f;
    }
    __syncthreads();
    const int groups = 256 / ct_n, rg = tid / ct_n, ct = tid - rg * ct_n;
    uint64_t qr[NQ][2], acc[NQ][2];
#pragma unroll
    for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = ct + 2 * h * ct_n;
            const float* o = qs + j * dp;
            qr[j][h] = packf(c < d ? o[few_at(c)] : 0.0f,
                             c + ct_n < d ? o[few_at(c + ct_n)] : 0.0f);
            acc[j][h] = 0ull;
        }
    int given[GIVEN ? NQ : 1];
#pragma unroll
    for (int e = 0; e < (GIVEN ? NQ : 0); ++e) {
        const int i = e * 256 + tid;
        given[e] = i < p.nq * p.given.k ? p.given.row[i] : -1;
    }
    // (unsigned: the last step may pass 2^31)
    for (unsigned u0 = blockIdx.x * FEW_ROWS; u0 < (unsigned)p.n; u0 += gridDim.x * FEW_ROWS) {
        const int r0 = (int)u0;
        {  // the next rows on their way
            const int lines = (d * (int)sizeof(T) + 127) / 128;
            for (int i = tid; i < FEW_ROWS * lines; i += 256) {
                const long long row = (long long)r0 + (long long)gridDim.x * FEW_ROWS + i / lines;
                if (row < p.n)
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(
                        p.x + (size_t)row * p.ldx + i % lines * (128 / (int)sizeof(T))));
            }
        }
        const int w0 = 2 * warp;
        if (lane < 2) x_bad[w0 + lane] = 0;
        const T* xa = p.x + (size_t)min(r0 + w0, p.n - 1) * p.ldx;
        const T* xb = p.x + (size_t)min(r0 + w0 + 1, p.n - 1) * p.ldx;
        uint64_t sa[NQ], sb[NQ];
#pragma unroll
        for (int j = 0; j < NQ; ++j) sa[j] = sb[j] = 0ull;
#pragma unroll 4
        for (int c = lane; c < d; c += 64) {
            const bool two = c + 32 < d;
            const T zero = from_f32<T>(0.0f);
            const T a0 = xa[c], b0 = xb[c];
            const T a1 = two ? xa[c + 32] : zero, b1 = two ? xb[c + 32] : zero;
            T* o = xs + w0 * dp + c;
            o[0] = a0, o[32] = a1, o[dp] = b0, o[dp + 32] = b1;
            const uint64_t a = packf(to_f32<T>(a0), to_f32<T>(a1));
            const uint64_t b = packf(to_f32<T>(b0), to_f32<T>(b1));
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
                const uint64_t v =
                    *reinterpret_cast<const uint64_t*>(qs + j * dp + (c & ~63) + 2 * lane);
                sa[j] = fma2(a, v, sa[j]);
                sb[j] = fma2(b, v, sb[j]);
            }
        }
        // halves of the sums are exchanged while more than one is left
        float v[2 * NQ];
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            v[2 * j] = lo_of(sa[j]) + hi_of(sa[j]);
            v[2 * j + 1] = lo_of(sb[j]) + hi_of(sb[j]);
        }
#pragma unroll
        for (int o = 16, m = NQ; o; o >>= 1, m >>= 1) {
            if (m > 0) {
#pragma unroll
                for (int i = 0; i < m; ++i) {
                    const float keep = lane & o ? v[i + m] : v[i];
                    const float give = lane & o ? v[i] : v[i + m];
                    v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                }
            } else {
                v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
            }
        }
        __syncwarp();
        if (lane % (16 / NQ) == 0) {
            const int i = lane / (16 / NQ), j = i >> 1, r = w0 + (i & 1), row = r0 + r;
            float g = 0.0f;
            if (j < p.nq && row < p.n) {
                const bool x_off = !(fabsf(v[0]) <= FLT_MAX);
                if (x_off) x_bad[r] = 1;
                const uint32_t w = allowed_word(p.coef.allowed, p.coef.ld_allowed, j,
                                                (size_t)(row & ~31), p.n);
                const Coef& k = co[j];
                const float y = __fmaf_rn(v[0], k.rf_hi, -k.l_hi) + __fmaf_rn(v[0], k.rf_lo, -k.l_lo);
                const float t = fmaxf(y, -160.0f);
                g = ex2(t) * __fmaf_rn(t, k.h, k.c);
                if (row == k.target) g += k.g;
                if (x_off || q_bad[j]) g = NAN;
                if (!(w >> (row & 31) & 1u)) g = 0.0f;
            }
            gs[r * NQ + j] = make_float2(g, g);
        }
        if (GIVEN) {
            bool here = false;
#pragma unroll
            for (int e = 0; e < NQ; ++e) here |= (unsigned)(given[e] - r0) < (unsigned)FEW_ROWS;
            if (__syncthreads_or(here)) {
#pragma unroll
                for (int e = 0; e < NQ; ++e)
                    if ((unsigned)(given[e] - r0) < (unsigned)FEW_ROWS) {
                        const int i = e * 256 + tid;
                        const float g = p.given.g[i];
                        gs[(given[e] - r0) * NQ + i / p.given.k] = make_float2(g, g);
                    }
                __syncthreads();
            }
        } else {
            __syncthreads();
        }
        if (rg < groups) {
#pragma unroll (NQ > 4 ? 1 : 2)
            for (int r = rg; r < FEW_ROWS; r += groups) {
                // (columns past the last: whatever lies there, for sums that nobody takes)
                const T* x = xs + r * dp + ct;
                float xv[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) xv[i] = to_f32<T>(x[i * ct_n]);
                if (r0 + r >= p.n) xv[0] = xv[1] = xv[2] = xv[3] = 0.0f;
                // (its elements, or only a product with a query that may not see it,
                // are not finite: the former reach those that see it through G)
                if (x_bad[r]) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!(fabsf(xv[i]) <= FLT_MAX)) xv[i] = 0.0f;
                }
                const uint64_t x2[2] = {packf(xv[0], xv[1]), packf(xv[2], xv[3])};
                uint64_t o2[2] = {0ull, 0ull};
#pragma unroll
                for (int j = 0; j < NQ; ++j) {
                    const uint64_t g2 = *reinterpret_cast<const uint64_t*>(gs + r * NQ + j);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        acc[j][h] = fma2(g2, x2[h], acc[j][h]);
                        o2[h] = fma2(g2, qr[j][h], o2[h]);
                    }
                }
                if (p.dx && r0 + r < p.n) {
                    T* o = p.dx + (size_t)(r0 + r) * p.ld_dx + ct;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float y = i & 1 ? hi_of(o2[i >> 1]) : lo_of(o2[i >> 1]);
                        if (ct + i * ct_n < d) o[i * ct_n] = from_f32<T>(y);
                    }
                }
            }
        }
        __syncthreads();
    }
    if (!p.partial) return;
    float* sums = reinterpret_cast<float*>(xs);  // [groups][NQ][4 ct_n]
    if (rg < groups) {
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                sums[(rg * NQ + j) * 4 * ct_n + ct + i * ct_n] =
                    i & 1 ? hi_of(acc[j][i >> 1]) : lo_of(acc[j][i >> 1]);
    }
    __syncthreads();
    for (int i = tid; i < p.nq * d; i += 256) {
        const int j = i / d, c = i - j * d;
        float t = 0.0f;
        for (int k = 0; k < min(groups, FEW_ROWS); ++k) t += sums[(k * NQ + j) * 4 * ct_n + c];
        p.partial[((size_t)blockIdx.x * p.nq + j) * d + c] = t;
    }
}
// A call whose waits ran out has no gradient: NaN.
__global__ void void_kernel(const int* err, void* dq, size_t ldq, int nq, void* dx, size_t ldx,
                            int n, int cols, int dtype) {
    wait_for_last();
    if (*err == 0) return;
    const size_t step = (size_t)gridDim.x * 256, i0 = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (dq)
        for (size_t i = i0; i < (size_t)nq * cols; i += step)
            put(dq, i / cols * ldq + i % cols, dtype, NAN);
    if (dx)
        for (size_t i = i0; i < (size_t)n * cols; i += step)
            put(dx, i / cols * ldx + i % cols, dtype, NAN);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
constexpr size_t HEAD = 256;                    // error word, GradHead
constexpr size_t CHUNK_BYTES = (size_t)512 << 20;  // of group maxima, of score gradients
// dims above which a score's sum is taken in blocks.  Whole sums are faster (2048 x
// 131072 x 768 bf16: 284 us) and stay while half of what a sum of one sign loses
// (see cut_of) is below 6e-7 of it: 768 bf16 (1.1e-6 in all), 256 f16 (0.8e-6).
// Two parts of 128 are one block: 4096 x 262144 x 96 f32 takes 811 us in tiles
// of 128 columns, 694 in those of 256, whose waits and loads serve twice as
// many.  The gradient's scores of 16-bit rows only have to be as good as G, which
// is held in 11 bits: at 1024 a score of 200 is off by 3.4e-4, less than the 4.9e-4
// that G is rounded by; above it would grow to 5e-3 at 16384 (1000 x 50001: 1024
// whole 328 us, in blocks 389; 2048 662 and 780).
constexpr size_t BLOCKS_F32 = 128, BLOCKS_F16 = 256, BLOCKS_BF16 = 768;
constexpr size_t BLOCKS_GRAD = 1024;
// Queries that few_kernel takes.  f32 rows would have to be split for the tensor
// cores first: 8 queries take 148 us here and 249 there (100000 x 768), 28 and 27
// (2000 x 128); 12, in two passes, 239 and 251, but 46 and 27.  16-bit rows are
// read by the tensor cores as they are, if their alignment lets a tensor map
// describe them (100000 x 376, 4 queries: 54 us here, 38 there), else after a copy
// (100000 x 374: 58 and 70, with 8 queries 79 and 69).
constexpr int FEW_F32 = 8, FEW_16 = 2, FEW_16_COPIED = 4, FEW_DIM = 2048;
// Queries and dimensions that few_grad_kernel takes (a call of 8: 100000 x 768 f32
// 261 us, by the tensor cores 486; bf16 259 and 265, 300000 x 96 171 and 239, 2000 x
// 128 19 and 56).
constexpr int FEW_GRAD = 8, FEW_GRAD_DIM = 1024;
static size_t smem_of(bool two, bool blk, bool grad) {
    // alignment, stages, staged outputs, barriers, column factors
    return 1024 + (size_t)stages_of(two, blk, grad) * stage_bytes(two, blk) +
           staged_of(two, grad) + 256 + EPI_WARPS * 128 * 4;
}

static void launch_align(cudaStream_t s, const void* x, size_t ld, size_t n, size_t d, size_t kp,
                         void* out) {
    // lanes for a row's 16-byte pieces: 8 to 32, so that the fewest are idle at its
    // end (300000 x 130: 27.6 us with 8, 49.2 with 32), 32 for 64 pieces and more
    // (50000 x 785: 39.5 and 30.8), fewer for shorter rows
    const size_t pieces = kp / 8;
    int shift = 0;
    while (shift < 3 && (size_t)1 << shift < pieces) ++shift;
    for (int i = 4; i <= 5; ++i)
        if (pieces >= 64 || up(pieces, (size_t)1 << i) <= up(pieces, (size_t)1 << shift)) shift = i;
    align_kernel<<<(unsigned)(((n << shift) + 255) / 256), 256, 0, s>>>(
        static_cast<const uint16_t*>(x), ld, (int)n, (int)d, (int)kp, shift,
        static_cast<uint16_t*>(out));
    FDB_LAUNCH_CHECK();
}
static size_t elem(int dtype) { return dtype == FDB_DTYPE_F32 ? 4 : 2; }

static CUtensorMap map2d(int dtype, const void* base, size_t inner, size_t rows, size_t ld_elems,
                         int box_rows, int box_cols = KATOM,
                         CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
    CUtensorMap m;
    cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld_elems * 2};
    cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
    cuuint32_t one[2] = {1, 1};
    const CUresult r = encode_fn()(
        &m,
        dtype == FDB_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
        2, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
        swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    FDB_REQUIRE(r == CUDA_SUCCESS, FDB_ERR_CUDA, "cuTensorMapEncodeTiled failed");
    return m;
}
// D f32; A and B both f16 or both bf16; transposed operands; M = 256 (N is added
// in the kernel).
static uint32_t idesc_of(int dtype, bool a_mn, bool b_mn) {
    const uint32_t t = dtype == FDB_DTYPE_BF16 ? 1u : 0u;
    return (1u << 4) | (t << 7) | (t << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
           ((uint32_t)(PM >> 4) << 24);
}
// Chunks of the column tiles: the count that leaves the busiest pair of blocks
// the fewest tiles, and of those the smallest.
static int pick_chunks(int mt, int nt, int sms) {
    sms = std::max(sms / 2, 1);
    int best = 1;
    long long cost = -1;
    for (int c = 1; c <= nt && c <= 4 * sms; ++c) {
        const long long waves = ((long long)mt * c + sms - 1) / sms;
        const long long t = waves * ((nt + c - 1) / c);
        if (cost < 0 || t < cost) cost = t, best = c;
    }
    return best;
}
// Splits of K of a rows x cols product.  A block runs the busiest share of the
// (tile, split) pairs at about 0.3 us per 64 of K (f32: 0.5); more than one
// split writes and reads `out_bytes` of partial sums each, at 4 MB/us, and
// takes another launch (3 us).
static int pick_splits(int tiles, int atoms, int sms, bool two, double out_bytes) {
    sms = std::max(sms / 2, 1);
    int best = 1;
    double cost = -1.0;
    for (int s = 1; s <= atoms && s <= 64; ++s) {
        const long long waves = ((long long)tiles * s + sms - 1) / sms;
        double t = (double)waves * ((atoms + s - 1) / s) * (two ? 0.5 : 0.3);
        if (s > 1) t += 3.0 + s * out_bytes * 2.0 / 4e6;
        if (cost < 0.0 || t < cost) cost = t, best = s;
    }
    return best;
}
static unsigned blocks_of(int sms, long long units) {
    return 2 * (unsigned)std::min<long long>(units, sms / 2);
}
template <int MODE, bool TWO, bool BLK>
static void launch_rows(bool over, cudaStream_t s, int device, int sms, const CUtensorMap& a,
                        const CUtensorMap& b, const Mma& g,
                        const typename EpilogueOf<MODE, TWO, BLK>::Type::Args& p,
                        const CUtensorMap* out = nullptr) {
    const long long units = MODE == PROD_Q || MODE == PROD_X
                                ? (long long)g.mt * g.nt * g.chunks
                                : (long long)g.mt * g.chunks;
    const size_t smem = smem_of(TWO, BLK, MODE == GRAD);
    static std::atomic<uint64_t> done{0};
    allow_smem(rows_kernel<MODE, TWO, BLK>, device, smem, done);
    launch(over, s, rows_kernel<MODE, TWO, BLK>, blocks_of(sms, units), THREADS, smem, a, b,
           out ? *out : a, g, p);
}
// A's K steps stay in shared memory where they fill at most half of the ring
// (4096 x 262144 x 96 f32: a tile's copies shrink to a third).
static int stays(bool two, bool blk, bool grad, int atoms) {
    return atoms * (two ? 2 : 1) * OPER <= stages_of(two, blk, grad) * stage_bytes(two, blk) / 2;
}
template <int MODE>
static void launch_product(bool two, cudaStream_t s, int device, int sms, const CUtensorMap& a,
                           const CUtensorMap& b, const Mma& g, const ProdArgs& p) {
    if (two) launch_rows<MODE, true, true>(true, s, device, sms, a, b, g, p);
    else launch_rows<MODE, false, false>(true, s, device, sms, a, b, g, p);
}

static PackSide pack_side(const void* x, size_t ld, size_t n, size_t dim, int dtype,
                          const uint32_t* seen, __half* out, float* f, unsigned* largest) {
    PackSide p{};
    p.x = x, p.ld = ld, p.n = (int)n, p.seen = seen, p.out = out, p.f = f, p.largest = largest;
    const size_t es = elem(dtype);
    p.wide = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ld * es & 15) == 0 &&
             (dim * es & 15) == 0;
    p.rows = dim * es <= 512 ? 4 : 1;
    p.blocks = (int)((n + 8 * p.rows - 1) / (8 * p.rows));
    return p;
}
static void launch_pack(bool over, cudaStream_t s, int dtype, const PackSide& a, const PackSide& b, size_t d,
                        size_t kp, int* err) {
    const auto kernel = dtype == FDB_DTYPE_F32   ? pack_kernel<float, 2>
                        : dtype == FDB_DTYPE_F16 ? pack_kernel<__half, 1>
                                                 : pack_kernel<__nv_bfloat16, 1>;
    launch(over, s, kernel, a.blocks + b.blocks, 256, 0, a, b, (int)d, (int)kp, err);
}

// The forward pass's workspace and launch shape.
struct Forward {
    bool few, packed, blocks, copy_q, copy_x;
    size_t kp, qb, groups, parts_cap;
    int bn, nt;
    size_t bytes;
    int* err;
    void *qp, *xp;
    float *qf, *xf;
    float4* part;
    float2* top;
    float* size;  // see FinishArgs
};
static bool mappable(const void* p, size_t ld) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * 2 & 15) == 0;
}
static Forward plan_forward(const Ctx& c, const fdb_logprob_args& a, size_t pass_queries) {
    Forward w{};
    Carve ws(a.workspace);
    w.err = ws.take<int>(HEAD / 4);
    w.few = a.nq <= (a.dtype == FDB_DTYPE_F32         ? FEW_F32
                     : mappable(a.rows, a.ld_rows) ? FEW_16
                                                   : FEW_16_COPIED) &&
            a.dim <= FEW_DIM;
    w.packed = a.dtype == FDB_DTYPE_F32 && !w.few;
    w.kp = up(a.dim, 16);
    // (sums in blocks where whole ones would lose over 1e-6 of a score)
    w.blocks = a.dim > (w.packed ? BLOCKS_F32 : a.dtype == FDB_DTYPE_F16 ? BLOCKS_F16 : BLOCKS_BF16);
    w.bn = bn_of(w.blocks);
    w.nt = (int)((a.n + w.bn - 1) / w.bn);
    w.groups = w.few ? (a.n + GROUP - 1) / GROUP : (size_t)w.nt * (w.bn / GROUP);
    const size_t per = a.k ? w.groups * sizeof(float2) : 0;
    w.qb = std::min<size_t>(a.nq, per ? std::max<size_t>(PM, CHUNK_BYTES / per / PM * PM)
                                      : (size_t)1 << 20);
    if (pass_queries) w.qb = std::min(w.qb, pass_queries);
    if (w.packed) {
        w.qp = ws.take<__half>(a.nq * 2 * w.kp);
        w.xp = ws.take<__half>(a.n * 2 * w.kp);
        w.qf = ws.take<float>(a.nq);
        w.xf = ws.take<float>((size_t)w.nt * w.bn);
    } else if (!w.few) {
        w.copy_q = !mappable(a.queries, a.ld_queries);
        w.copy_x = !mappable(a.rows, a.ld_rows);
        if (w.copy_q) w.qp = ws.take<__half>(a.nq * w.kp);
        if (w.copy_x) w.xp = ws.take<__half>(a.n * w.kp);
    }
    if (w.few) {
        w.parts_cap = std::min<size_t>((w.groups + 1) / 2, (size_t)c.sm_count * 12);
    } else {
        // (the last pass has fewer row blocks and may take more chunks)
        const int full = (int)((w.qb + PM - 1) / PM);
        const int last = (int)((a.nq % w.qb + PM - 1) / PM);
        w.parts_cap = 4 * (size_t)pick_chunks(full, w.nt, c.sm_count);
        if (last && last != full)
            w.parts_cap = std::max(w.parts_cap, 4 * (size_t)pick_chunks(last, w.nt, c.sm_count));
    }
    w.part = ws.take<float4>(w.parts_cap * w.qb);
    if (a.k) w.top = ws.take<float2>(w.qb * w.groups);
    if (a.k && (w.few || w.packed))
        w.size = ws.take<float>(std::max<size_t>(w.parts_cap, c.sm_count));
    w.bytes = ws.at;
    return w;
}
size_t forward_bytes(const Ctx& c, const fdb_logprob_args& a, size_t pass_queries) {
    fdb_logprob_args b = a;
    b.workspace = nullptr;
    return plan_forward(c, b, pass_queries).bytes;
}

template <typename T, int THREADS_>
static void launch_finish_t(cudaStream_t s, int device, const FinishArgs& f) {
    const size_t smem = (size_t)f.d * sizeof(typename Exact<T>::Q);
    if (smem > 4096) {  // (with the static part, over what needs no permission)
        static std::atomic<uint64_t> done{0};
        allow_smem(finish_kernel<T, THREADS_>, device,
                   FDB_MAX_SOFTMAX_DIM * sizeof(typename Exact<T>::Q), done);
    }
    finish_kernel<T, THREADS_><<<f.nq, THREADS_, smem, s>>>(f);
    FDB_LAUNCH_CHECK();
}
template <typename T>
static void launch_finish(cudaStream_t s, int device, const FinishArgs& f) {
    // A block a query.  Few queries: more threads share the groups of one.
    if (f.nq <= 296) launch_finish_t<T, 512>(s, device, f);
    else launch_finish_t<T, 128>(s, device, f);
}

// The share of a score that the tensor core's additions cut off on average,
// for sums over `block` 16-wide steps (0: all of them).  They cut towards zero:
// terms of one sign fall short by a share of the score that grows with the steps
// (measured over rows of 16 to 768 dimensions: 5.2e-8 a step less 2e-8 for fp16
// products, 2.3e-8 a step for bf16, with a spread of 0.6 to 1.0e-7 between
// scores), in sums of mixed signs nearly all of it cancels.  Half of the former
// is added to every score, so that neither kind is off by more than half.
static double cut_of(bool bf16, size_t dim, int block) {
    const double steps = (double)((dim + 15) / 16), b = block ? block : steps;
    auto cut = [&](double n) { return bf16 ? 2.3e-8 * n : 5.2e-8 * n - 2e-8; };
    const double whole = floor(steps / b) * b, rest = steps - whole;
    return 0.5 * (whole * cut(b) + (rest > 0.0 ? rest * cut(rest) : 0.0)) / steps;
}
static FinishArgs finish_args(const fdb_logprob_args& a, const Forward& w, size_t q0, size_t nq) {
    FinishArgs f{};
    f.q = a.queries, f.x = a.rows;
    f.ldq = a.ld_queries, f.ldx = a.ld_rows;
    f.q0 = (int)q0, f.nq = (int)nq, f.n = (int)a.n, f.d = (int)a.dim, f.k = (int)a.k;
    f.scale = a.scale;
    f.targets = a.targets;
    f.allowed = a.allowed, f.ld_allowed = a.allowed ? a.ld_allowed : 0;
    f.part = w.part;
    f.top = w.top, f.groups = w.groups;
    f.size = w.size, f.xf = w.xf;
    f.logprob = a.logprob, f.lse = a.lse, f.entropy = a.entropy;
    f.top_logprob = a.top_logprobs, f.top_ids = a.top_ids;
    f.err = w.err;
    f.whole = w.few ? 1.0
                    : 1.0 + cut_of(a.dtype == FDB_DTYPE_BF16, a.dim,
                                   w.blocks ? 4 * kblock_of(w.packed, false) : 0);
    return f;
}

static Parts parts_of(const FinishArgs& f) {
    return Parts{f.part, f.parts, f.q0, f.nq, f.qf, f.whole, f.err};
}
template <typename T, int NQ, bool VEC, bool TOP>
static void launch_few(const Ctx& c, const fdb_logprob_args& a, const Forward& w, float rf,
                       size_t ld_allowed) {
    const size_t smem = NQ * up(a.dim, 128) * 4;
    if (smem > 40960) {  // (with the static part, over what needs no permission)
        static std::atomic<uint64_t> done{0};
        allow_smem(few_kernel<T, NQ, VEC, TOP>, c.device, NQ * up(FEW_DIM, 128) * 4, done);
    }
    few_kernel<T, NQ, VEC, TOP><<<(unsigned)w.parts_cap, 64, smem, static_cast<cudaStream_t>(a.stream)>>>(
        static_cast<const T*>(a.rows), a.ld_rows, (int)a.n, (int)a.dim,
        static_cast<const T*>(a.queries), a.ld_queries, (int)a.nq, rf, a.allowed, ld_allowed, w.part,
        w.top, w.groups, w.size, w.err);
    FDB_LAUNCH_CHECK();
}
template <typename T, int NQ, bool VEC>
static void launch_few(const Ctx& c, const fdb_logprob_args& a, const Forward& w, float rf,
                       size_t ld_allowed) {
    if (w.top) launch_few<T, NQ, VEC, true>(c, a, w, rf, ld_allowed);
    else launch_few<T, NQ, VEC, false>(c, a, w, rf, ld_allowed);
}
template <typename T, int NQ>
static void launch_few(bool vec, const Ctx& c, const fdb_logprob_args& a, const Forward& w,
                       float rf, size_t ld_allowed) {
    if (vec) launch_few<T, NQ, true>(c, a, w, rf, ld_allowed);
    else launch_few<T, NQ, false>(c, a, w, rf, ld_allowed);
}
template <typename T>
static void few_run(const Ctx& c, const fdb_logprob_args& a, const Forward& w, float rf,
                    size_t ld_allowed, ForwardEnd* end) {
    const cudaStream_t s = static_cast<cudaStream_t>(a.stream);
    const bool vec = (reinterpret_cast<uintptr_t>(a.rows) & 15) == 0 &&
                     a.ld_rows * sizeof(T) % 16 == 0 && a.dim * sizeof(T) % 16 == 0;
    if (a.nq == 1) launch_few<T, 1>(vec, c, a, w, rf, ld_allowed);
    else if (a.nq == 2) launch_few<T, 2>(vec, c, a, w, rf, ld_allowed);
    else if constexpr (sizeof(T) == 4) {
        if (a.nq <= 4) launch_few<T, 4>(vec, c, a, w, rf, ld_allowed);
        else launch_few<T, 8>(vec, c, a, w, rf, ld_allowed);
    } else {  // (more than FEW_16: rows that would be copied, so unaligned ones)
        launch_few<T, 4, false>(c, a, w, rf, ld_allowed);
    }
    FinishArgs f = finish_args(a, w, 0, a.nq);
    f.parts = f.sizes = (int)w.parts_cap;
    if (end) end->finish(parts_of(f));
    else launch_finish<T>(s, c.device, f);
}

void forward_run(Ctx& c, const fdb_logprob_args& given, ForwardEnd* end) {
    fdb_logprob_args a = given;
    const cudaStream_t s = static_cast<cudaStream_t>(a.stream);
    const Forward w = plan_forward(c, a, end ? end->queries : 0);
    // (few queries are one pass)
    const bool filters = end && a.allowed && a.ld_allowed;
    if (filters && w.few) a.allowed = end->filters(0, a.nq, false);
    const int n = (int)a.n, d = (int)a.dim;
    const float rf = (float)((double)a.scale * LOG2E);
    const size_t ld_allowed = a.allowed ? a.ld_allowed : 0;
    Mma g{};
    CUtensorMap amap, bmap;
    if (!w.few) {
        if (!w.packed) FDB_CUDA(cudaMemsetAsync(w.err, 0, 4, s));
        const void *qb = a.queries, *xb = a.rows;
        size_t ldq = a.ld_queries, ldx = a.ld_rows, inner = a.dim;
        if (w.packed) {
            launch_pack(false, s, a.dtype,
                        pack_side(a.queries, a.ld_queries, a.nq, a.dim, a.dtype, nullptr,
                                  static_cast<__half*>(w.qp), w.qf, nullptr),
                        pack_side(a.rows, a.ld_rows, a.n, a.dim, a.dtype, nullptr,
                                  static_cast<__half*>(w.xp), w.xf, nullptr),
                        a.dim, w.kp, w.err);
            qb = w.qp, xb = w.xp;
            ldq = ldx = inner = 2 * w.kp;
        }
        if (w.copy_q) {
            launch_align(s, a.queries, a.ld_queries, a.nq, a.dim, w.kp, w.qp);
            qb = w.qp, ldq = w.kp;
        }
        if (w.copy_x) {
            launch_align(s, a.rows, a.ld_rows, a.n, a.dim, w.kp, w.xp);
            xb = w.xp, ldx = w.kp;
        }
        bmap = map2d(a.dtype, xb, inner, a.n, ldx, w.bn / 2);
        g.nt = w.nt;
        g.atoms = (int)((w.kp + 63) / 64);
        g.klast = (int)((w.kp - 64 * (size_t)(g.atoms - 1)) / 16);
        g.resident = stays(w.packed, w.blocks, false, g.atoms);
        g.a_part = g.b_part = (int)w.kp;
        g.idesc = idesc_of(w.packed ? FDB_DTYPE_F16 : a.dtype, false, false);
        g.err = w.err;
        g.wait = wait_limit_cycles(c);
        g.stall = take_test_stall(c);
        for (size_t q0 = 0; q0 < a.nq; q0 += w.qb) {
            const size_t nq = std::min(w.qb, a.nq - q0);
            g.mt = (int)((nq + PM - 1) / PM);
            g.chunks = pick_chunks(g.mt, w.nt, c.sm_count);
            amap = map2d(a.dtype,
                         static_cast<const unsigned char*>(qb) + q0 * ldq * 2, inner, nq, ldq, BM);
            StatsArgs p{};
            p.q0 = filters ? 0 : (int)q0;  // (counts for the filters alone)
            p.nq = (int)nq;
            p.n = n;
            p.qf = w.packed ? w.qf + q0 : nullptr;
            p.xf = w.xf;
            p.rf = rf;
            bool over = q0 > 0 || w.packed || w.copy_q || w.copy_x;
            p.allowed = filters ? end->filters(q0, nq, over) : a.allowed;
            over |= filters;
            p.ld_allowed = ld_allowed;
            p.part = w.part;
            p.top = w.top;
            p.groups = w.groups;
            p.size = w.size;
            if (w.packed && !w.blocks)
                launch_rows<STATS, true, false>(over, s, c.device, c.sm_count, amap, bmap, g, p);
            else if (w.packed)
                launch_rows<STATS, true, true>(over, s, c.device, c.sm_count, amap, bmap, g, p);
            else if (w.blocks)
                launch_rows<STATS, false, true>(over, s, c.device, c.sm_count, amap, bmap, g, p);
            else
                launch_rows<STATS, false, false>(over, s, c.device, c.sm_count, amap, bmap, g, p);
            FinishArgs f = finish_args(a, w, q0, nq);
            f.parts = g.chunks * 4;
            f.qf = p.qf;
            f.sizes = (int)blocks_of(c.sm_count, (long long)g.mt * g.chunks);
            f.nt = w.nt, f.chunks = g.chunks;
            f.per_tile = w.bn / GROUP, f.per_part = w.bn / GROUP / 4;
            if (end) end->finish(parts_of(f));
            else if (a.dtype == FDB_DTYPE_F32) launch_finish<float>(s, c.device, f);
            else if (a.dtype == FDB_DTYPE_F16) launch_finish<__half>(s, c.device, f);
            else launch_finish<__nv_bfloat16>(s, c.device, f);
        }
        return;
    }
    if (a.dtype == FDB_DTYPE_F32) few_run<float>(c, a, w, rf, ld_allowed, end);
    else if (a.dtype == FDB_DTYPE_F16) few_run<__half>(c, a, w, rf, ld_allowed, end);
    else few_run<__nv_bfloat16>(c, a, w, rf, ld_allowed, end);
}

// ---- backward ----
struct Backward {
    bool few;
    int parts, few_blocks;
    size_t kp, nqp, cols, ldg;  // cols: rows of a chunk
    bool blocks;                // GRAD's sums
    int bn, q_splits, x_splits;
    size_t bytes;
    int* err;
    GradHead* head;
    __half *qp, *qs, *xp, *gr;
    float *qf, *xf, *out_f, *dq, *dx;
    int* weight;
    Coef* coef;
    float* rest;
    int* rest_row;
    uint32_t *seen, *alive;
};
static Backward plan_backward(const Ctx& c, const fdb_logprob_grad_args& a, const GivenRows* given) {
    Backward w{};
    Carve ws(a.workspace);
    w.few = a.nq <= FEW_GRAD && a.dim <= FEW_GRAD_DIM;
    if (w.few) {
        w.err = ws.take<int>(HEAD / 4);
        w.few_blocks = (int)std::min<size_t>((a.n + FEW_ROWS - 1) / FEW_ROWS,
                                             few_per_sm((int)a.nq) * c.sm_count);
        w.dq = ws.take<float>((size_t)w.few_blocks * a.nq * a.dim);
        w.bytes = ws.at;
        return w;
    }
    w.parts = a.dtype == FDB_DTYPE_F32 ? 2 : 1;
    w.kp = up(a.dim, 16);
    w.nqp = up(a.nq, BM);
    w.blocks = w.parts == 2 || a.dim > BLOCKS_GRAD;
    w.bn = bn_of(w.parts == 2);
    const size_t row_bytes = w.nqp * 2 * w.parts;
    w.cols = std::min<size_t>(std::max<size_t>(MAX_BN, CHUNK_BYTES / row_bytes / MAX_BN * MAX_BN),
                              a.n);
    w.ldg = up(w.cols, 64);
    const int ntd = (int)((a.dim + w.bn - 1) / w.bn);
    w.q_splits = pick_splits((int)((a.nq + PM - 1) / PM) * ntd, (int)((w.cols + 63) / 64), c.sm_count,
                             w.parts == 2, (double)a.nq * a.dim * 4);
    w.x_splits = pick_splits((int)((w.cols + PM - 1) / PM) * ntd, (int)((a.nq + 63) / 64),
                             c.sm_count, w.parts == 2, (double)w.cols * a.dim * 4);
    unsigned char* head = ws.take<unsigned char>(HEAD);
    w.err = reinterpret_cast<int*>(head);
    w.head = reinterpret_cast<GradHead*>(head ? head + 64 : nullptr);
    w.qp = ws.take<__half>(a.nq * w.parts * w.kp);
    w.qs = ws.take<__half>(a.nq * w.parts * w.kp);
    w.xp = ws.take<__half>(a.n * w.parts * w.kp);
    w.qf = ws.take<float>(a.nq);
    w.xf = ws.take<float>(up(a.n, MAX_BN) + MAX_BN);
    w.out_f = ws.take<float>(a.nq);
    w.weight = ws.take<int>(a.nq);
    w.coef = ws.take<Coef>(a.nq);
    if (w.parts == 1) w.rest = ws.take<float>(a.nq);
    if (w.parts == 1 && given) w.rest_row = ws.take<int>(a.nq);
    w.gr = ws.take<__half>((size_t)w.parts * w.nqp * w.ldg);
    w.dq = ws.take<float>((size_t)w.q_splits * a.nq * a.dim);
    if (w.x_splits > 1) w.dx = ws.take<float>((size_t)w.x_splits * w.cols * a.dim);
    w.alive = ws.take<uint32_t>((a.nq + 31) / 32);
    if (a.allowed && a.ld_allowed) w.seen = ws.take<uint32_t>((a.n + 31) / 32);
    w.bytes = ws.at;
    return w;
}
size_t backward_bytes(const Ctx& c, const fdb_logprob_grad_args& a, const GivenRows* given) {
    fdb_logprob_grad_args b = a;
    b.workspace = nullptr;
    return plan_backward(c, b, given).bytes;
}

BackwardHead backward_head(const Ctx& c, const fdb_logprob_grad_args& a, const GivenRows& given) {
    const Backward w = plan_backward(c, a, &given);
    if (w.few) return BackwardHead{};
    return BackwardHead{w.weight, reinterpret_cast<uint32_t*>(w.err), (int)(HEAD / 4)};
}

template <typename T, int NQ, bool GIVEN>
static void launch_few_grad(const Ctx& c, const Backward& w, const FewGrad<T>& p, cudaStream_t s) {
    const size_t smem = few_grad_smem(NQ, p.d, sizeof(T));
    if (smem > 40960) {  // (see allow_smem)
        static std::atomic<uint64_t> done{0};
        allow_smem(few_grad_kernel<T, NQ, GIVEN>, c.device,
                   few_grad_smem(NQ, FEW_GRAD_DIM, sizeof(T)), done);
    }
    launch(GIVEN, s, few_grad_kernel<T, NQ, GIVEN>, w.few_blocks, 256, smem, p);
}
template <typename T, bool GIVEN>
static void launch_few_grad(const Ctx& c, const Backward& w, const FewGrad<T>& p, cudaStream_t s) {
    if (p.nq == 1) launch_few_grad<T, 1, GIVEN>(c, w, p, s);
    else if (p.nq == 2) launch_few_grad<T, 2, GIVEN>(c, w, p, s);
    else if (p.nq <= 4) launch_few_grad<T, 4, GIVEN>(c, w, p, s);
    else launch_few_grad<T, 8, GIVEN>(c, w, p, s);
}
template <typename T>
static void few_backward(const Ctx& c, const fdb_logprob_grad_args& a, const Backward& w,
                         const CoefArgs& k, const GivenRows* given) {
    const cudaStream_t s = static_cast<cudaStream_t>(a.stream);
    FewGrad<T> p{};
    p.x = static_cast<const T*>(a.rows), p.ldx = a.ld_rows;
    p.q = static_cast<const T*>(a.queries), p.ldq = a.ld_queries;
    p.n = (int)a.n, p.d = (int)a.dim, p.nq = (int)a.nq;
    p.coef = k;
    p.dx = static_cast<T*>(a.d_rows), p.ld_dx = a.ld_d_rows;
    p.partial = a.d_queries ? w.dq : nullptr;
    p.err = w.err;
    if (given) {
        p.given = *given;
        launch_few_grad<T, true>(c, w, p, s);
    } else {
        launch_few_grad<T, false>(c, w, p, s);
    }
    if (a.d_queries)
        launch_join(s, c.sm_count, w.dq, w.few_blocks, (int)a.nq, (int)a.dim, nullptr, nullptr,
                    a.d_queries, a.ld_d_queries, a.dtype);
}

void backward_run(Ctx& c, const fdb_logprob_grad_args& a, const GivenRows* given) {
    const cudaStream_t s = static_cast<cudaStream_t>(a.stream);
    const Backward w = plan_backward(c, a, given);
    if (w.few) {
        CoefArgs k{};
        k.nq = (int)a.nq, k.n = (int)a.n, k.scale = a.scale, k.whole = 1.0;
        k.lse = a.lse, k.entropy = a.entropy;
        k.d_logprob = a.d_logprob, k.d_lse = a.d_lse, k.d_entropy = a.d_entropy;
        k.targets = a.targets, k.allowed = a.allowed, k.ld_allowed = a.allowed ? a.ld_allowed : 0;
        if (a.dtype == FDB_DTYPE_F32) few_backward<float>(c, a, w, k, given);
        else if (a.dtype == FDB_DTYPE_F16) few_backward<__half>(c, a, w, k, given);
        else few_backward<__nv_bfloat16>(c, a, w, k, given);
        return;
    }
    const int n = (int)a.n, d = (int)a.dim, nq = (int)a.nq;
    const size_t ld_allowed = a.allowed ? a.ld_allowed : 0;
    CoefArgs k{};
    k.nq = nq, k.n = n, k.scale = a.scale;
    k.whole = 1.0 + cut_of(false, a.dim, w.blocks ? 4 * kblock_of(w.parts == 2, true) : 0);
    k.lse = a.lse, k.entropy = a.entropy;
    k.d_logprob = a.d_logprob, k.d_lse = a.d_lse, k.d_entropy = a.d_entropy;
    k.targets = a.targets, k.allowed = a.allowed, k.ld_allowed = ld_allowed;
    k.out = w.coef, k.rest = w.rest;
    if (given) k.at_least = given->at_least;
    if (!given) {
        head_kernel<<<(nq + 63) / 64, 64, 0, s>>>(k, w.alive, w.weight,
                                                     reinterpret_cast<uint32_t*>(w.err), HEAD / 4);
        FDB_LAUNCH_CHECK();
    }
    const uint32_t* seen = a.allowed;
    if (w.seen) {
        const size_t words = (a.n + 31) / 32;
        launch(true, s, any_kernel, (words + 31) / 32, 1024, 0, a.allowed, a.ld_allowed, nq, words,
               w.seen);
        seen = w.seen;
    }
    PackSide qside = pack_side(a.queries, a.ld_queries, a.nq, a.dim, a.dtype, w.alive, w.qp, w.qf,
                               &w.head->q_most);
    qside.weight = w.weight;
    if (given) qside.seen = nullptr, qside.lse = a.lse;
    launch_pack(true, s, a.dtype, qside,
                pack_side(a.rows, a.ld_rows, a.n, a.dim, a.dtype, seen, w.xp, w.xf,
                          reinterpret_cast<unsigned*>(&w.head->x_most)),
                a.dim, w.kp, nullptr);
    const int qblocks = (nq + 7) / 8;
    launch(true, s, settle_kernel, qblocks + (n + 255) / 256, 256, 0, k, w.qp, w.qf, w.weight, w.qs,
           w.out_f, w.xp, w.xf, (int)w.kp, w.parts, qblocks, w.head);

    const size_t width = w.parts * w.kp;
    const bool two = w.parts == 2;
    const int mtq = (int)((a.nq + PM - 1) / PM), ntd = (d + w.bn - 1) / w.bn;
    const CUtensorMap qk = map2d(FDB_DTYPE_F16, w.qp, width, a.nq, width, BM);
    const int grad_bn = bn_of(w.blocks);
    const CUtensorMap xk = map2d(FDB_DTYPE_F16, w.xp, width, a.n, width, grad_bn / 2);
    const CUtensorMap qm = map2d(FDB_DTYPE_F16, w.qs, width, a.nq, width, 64);
    const CUtensorMap xm = map2d(FDB_DTYPE_F16, w.xp, width, a.n, width, 64);
    const size_t g_rows = w.parts * w.nqp;
    const CUtensorMap gk = map2d(FDB_DTYPE_F16, w.gr, w.ldg, g_rows, w.ldg, BM);
    const CUtensorMap gm = map2d(FDB_DTYPE_F16, w.gr, w.ldg, g_rows, w.ldg, 64);
    const CUtensorMap go = map2d(FDB_DTYPE_F16, w.gr, w.ldg, g_rows, w.ldg, 32, 32,
                                 CU_TENSOR_MAP_SWIZZLE_64B);
    Mma base{};
    base.err = w.err;
    base.wait = wait_limit_cycles(c);
    base.stall = take_test_stall(c);
    for (size_t j0 = 0; j0 < a.n; j0 += w.cols) {
        const int cols = (int)std::min(w.cols, a.n - j0);
        {
            Mma g = base;
            g.mt = mtq;
            g.nt = (cols + grad_bn - 1) / grad_bn;
            g.chunks = pick_chunks(g.mt, g.nt, c.sm_count);
            g.atoms = (int)((w.kp + 63) / 64);
            g.klast = (int)((w.kp - 64 * (size_t)(g.atoms - 1)) / 16);
            g.resident = stays(two, w.blocks, true, g.atoms);
            g.a_part = g.b_part = (int)w.kp;
            g.b_row0 = (int)j0;
            g.idesc = idesc_of(FDB_DTYPE_F16, false, false);
            GradArgs p{};
            p.nq = nq, p.n = n, p.j0 = (int)j0, p.cols = cols;
            p.coef = w.coef, p.xf = w.xf;
            p.allowed = a.allowed, p.ld_allowed = ld_allowed;
            p.ldg = w.ldg, p.nqp = (int)w.nqp, p.rest = w.rest;
            if (two) launch_rows<GRAD, true, true>(true, s, c.device, c.sm_count, qk, xk, g, p, &go);
            else if (w.blocks)
                launch_rows<GRAD, false, true>(true, s, c.device, c.sm_count, qk, xk, g, p, &go);
            else launch_rows<GRAD, false, false>(true, s, c.device, c.sm_count, qk, xk, g, p, &go);
        }
        if (given) {
            const GivenArgs p{*given, nq, w.weight, w.xf, w.gr, w.ldg, (int)w.nqp, w.parts,
                              (int)j0, cols, j0 == 0 ? w.rest : nullptr, w.rest_row};
            launch(true, s, given_kernel, (nq + 7) / 8, 256, 0, p);
        }
        if (a.d_queries) {
            Mma g = base;
            g.mt = mtq, g.nt = ntd;
            g.atoms = (cols + 63) / 64;
            g.klast = 4;
            g.chunks = std::min(w.q_splits, g.atoms);
            g.a_part = (int)w.nqp, g.b_part = (int)w.kp;
            g.b_row0 = (int)j0;
            g.ncols = d;
            g.idesc = idesc_of(FDB_DTYPE_F16, false, true);
            ProdArgs p{};
            p.rows = nq, p.cols = d, p.f = w.out_f;
            p.partial = w.dq, p.add = j0 > 0;
            launch_product<PROD_Q>(two, s, c.device, c.sm_count, gk, xm, g, p);
        }
        if (a.d_rows) {
            Mma g = base;
            g.mt = (cols + PM - 1) / PM, g.nt = ntd, g.chunks = w.x_splits;
            g.atoms = (nq + 63) / 64;
            g.klast = 4;
            g.a_part = (int)w.nqp, g.b_part = (int)w.kp;
            g.ncols = d;
            g.idesc = idesc_of(FDB_DTYPE_F16, true, true);
            unsigned char* out =
                static_cast<unsigned char*>(a.d_rows) + j0 * a.ld_d_rows * elem(a.dtype);
            ProdArgs p{};
            p.rows = cols, p.cols = d, p.f = w.xf + j0, p.head = w.head;
            p.partial = w.dx;
            p.out = out, p.ldo = a.ld_d_rows, p.dtype = a.dtype;
            launch_product<PROD_X>(two, s, c.device, c.sm_count, gm, qm, g, p);
            if (w.dx) {
                launch_join(s, c.sm_count, w.dx, w.x_splits, cols, d, w.xf + j0, w.head, out,
                            a.ld_d_rows, a.dtype);
            }
        }
    }
    if (a.d_queries) {
        JoinRest rest{w.rest, w.rest_row, 1, w.xp, (int)width};
        if (!given) rest.row = &w.coef->target, rest.step = sizeof(Coef) / sizeof(int);
        launch_join(s, c.sm_count, w.dq, w.q_splits, nq, d, w.out_f, nullptr, a.d_queries,
                    a.ld_d_queries, a.dtype, rest);
    }
    launch(true, s, void_kernel, c.sm_count, 256, 0, w.err, a.d_queries, a.ld_d_queries, nq, a.d_rows,
           a.ld_d_rows, n, d, a.dtype);
}

// One thread per row: its id among the sorted wanted ones, the lowest row kept.
__global__ void find_rows_kernel(const uint64_t* __restrict__ ids, size_t n,
                                 const uint64_t* __restrict__ sorted, size_t count,
                                 unsigned long long* __restrict__ slot) {
    const size_t j = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (j >= n) return;
    const uint64_t id = ids[j];
    size_t lo = 0, hi = count;
    while (lo < hi) {
        const size_t mid = (lo + hi) >> 1;
        if (sorted[mid] < id) lo = mid + 1;
        else hi = mid;
    }
    if (lo < count && sorted[lo] == id) atomicMin(slot + lo, (unsigned long long)j);
}
void launch_find_rows(cudaStream_t s, const uint64_t* ids, size_t n, const uint64_t* sorted,
                      size_t count, unsigned long long* slot) {
    find_rows_kernel<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(ids, n, sorted, count, slot);
    FDB_LAUNCH_CHECK();
}

}  // namespace sr
}  // namespace fdb
