// beam.cu -- one step of a beam search: the best continuations over beams and
// columns, and states that follow the beams they were taken from.
//
//   l_bj = scale x_bj - log sum_j exp(scale x_bj)   (or scale x_bj)
//   the `width` largest beam_b + l_bj, equal ones by beam, then column
//
// Scores are compared in 64 bits, as a 32-bit sum of two of them would make equal
// what is not.
#include <cmath>

#include "softmax_rows.cuh"

namespace fdb {
namespace beam {

using sr::Carve;
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
    double* lse;  // [chains]
};

// scale x of a column, -inf if it takes no part
template <typename T>
__device__ __forceinline__ double column(const Select& p, int g, int b, int j) {
    const size_t row = (size_t)g * p.beams + b;
    if (p.ids && p.ids[row * p.ld_ids + j] < 0) return -INFINITY;
    if (p.allowed && !(p.allowed[row * p.ld_allowed + (j >> 5)] >> (j & 31) & 1u)) return -INFINITY;
    const T* x = static_cast<const T*>(p.x) + (size_t)g * p.ld_group + (size_t)b * p.ld_beam;
    return p.scale * (double)to_f32<T>(x[j]);
}
__device__ __forceinline__ bool over(const Select& p, int g, int b) {
    return p.ended && p.ended[(size_t)g * p.beams + b];
}
// A chain that is not there: whatever its columns hold.
__device__ __forceinline__ bool absent(const Select& p, int g, int b) {
    return p.beam_scores[(size_t)g * p.beams + b] == -INFINITY;
}

// One block per chain: its normaliser (0 without), NaN if a column that takes part
// is NaN or +inf.
template <typename T>
__global__ void __launch_bounds__(256) lse_kernel(const Select p) {
    __shared__ double part[8];
    const int g = blockIdx.x / p.beams, b = blockIdx.x % p.beams;
    if (over(p, g, b) || absent(p, g, b)) return;
    double m = -INFINITY;
    bool bad = false;
    for (int j = threadIdx.x; j < p.n; j += 256) {
        const double v = column<T>(p, g, b, j);
        bad |= !(v < INFINITY);
        m = fmax(m, v);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    bad = __syncthreads_or(bad);
    for (int i = 0; i < 8; ++i) m = fmax(m, part[i]);
    __syncthreads();
    double s = 0.0;
    if (p.normalise && !bad && m > -INFINITY)
        for (int j = threadIdx.x; j < p.n; j += 256) s += exp(column<T>(p, g, b, j) - m);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x != 0) return;
    s = 0.0;
    for (int i = 0; i < 8; ++i) s += part[i];
    p.lse[blockIdx.x] = bad ? NAN : m == -INFINITY || !p.normalise ? 0.0 : m + log(s);
}

// One block per search: the best candidate after the one before, `width` times.
template <typename T>
__global__ void __launch_bounds__(1024) pick_kernel(const Select p) {
    __shared__ double best_s[32];
    __shared__ unsigned long long best_at[32];
    const int g = blockIdx.x, tid = threadIdx.x;
    bool bad = false;
    for (int b = tid; b < p.beams; b += 1024) {
        const float s = p.beam_scores[(size_t)g * p.beams + b];
        bad |= !(s < INFINITY);
        if (!over(p, g, b) && !absent(p, g, b)) bad |= !(p.lse[(size_t)g * p.beams + b] < INFINITY);
    }
    bad = __syncthreads_or(bad);
    double last = INFINITY;
    unsigned long long last_at = 0;
    for (int w = 0; w < p.width; ++w) {
        double s = -INFINITY;
        unsigned long long at = ~0ull;
        for (int b = 0; b < p.beams && !bad; ++b) {
            const double sum = p.beam_scores[(size_t)g * p.beams + b];
            if (absent(p, g, b)) continue;
            const bool done = over(p, g, b);
            const double lse = done ? 0.0 : p.lse[(size_t)g * p.beams + b];
            for (int j = tid; j < (done ? 1 : p.n); j += 1024) {
                const double v = done ? sum : sum + (column<T>(p, g, b, j) - lse);
                const unsigned long long a = (unsigned long long)b << 32 | (unsigned)j;
                if (v > last || (v == last && a <= last_at && w)) continue;
                if (v > s || (v == s && a < at)) s = v, at = a;
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const double os = __shfl_xor_sync(0xffffffffu, s, o);
            const unsigned long long oa = __shfl_xor_sync(0xffffffffu, at, o);
            if (os > s || (os == s && oa < at)) s = os, at = oa;
        }
        __syncthreads();
        if ((tid & 31) == 0) best_s[tid >> 5] = s, best_at[tid >> 5] = at;
        __syncthreads();
        for (int i = 0; i < 32; ++i)
            if (best_s[i] > s || (best_s[i] == s && best_at[i] < at)) s = best_s[i], at = best_at[i];
        last = s, last_at = at;
        if (tid != 0) continue;
        const size_t o = (size_t)g * p.width + w;
        const bool none = bad || s == -INFINITY;
        const int b = (int)(at >> 32), j = (int)(at & 0x7fffffffu);
        const bool done = !none && over(p, g, b);
        int64_t id = -1;
        if (!none)
            id = done ? p.end_id : p.ids ? p.ids[((size_t)g * p.beams + b) * p.ld_ids + j] : j;
        p.out_scores[o] = bad ? NAN : (float)s;
        p.out_parents[o] = none ? -1 : b;
        p.out_ids[o] = id;
        if (p.out_ended) p.out_ended[o] = !none && (done || id == p.end_id);
    }
}

static size_t plan(const fdb_beam_args& a, Select* p) {
    Carve ws(a.workspace);
    double* lse = ws.take<double>(a.groups * a.beams);
    if (p) p->lse = lse;
    return ws.at;
}
size_t select_bytes(const Ctx&, const fdb_beam_args& a) { return plan(a, nullptr); }

template <typename T>
static void run(const fdb_beam_args& a, const Select& p) {
    const cudaStream_t s = static_cast<cudaStream_t>(a.stream);
    lse_kernel<T><<<(unsigned)(a.groups * a.beams), 256, 0, s>>>(p);
    FDB_LAUNCH_CHECK();
    pick_kernel<T><<<(unsigned)a.groups, 1024, 0, s>>>(p);
    FDB_LAUNCH_CHECK();
}
void select_run(const Ctx&, const fdb_beam_args& a) {
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
    plan(a, &p);
    if (a.dtype == FDB_DTYPE_F32) run<float>(a, p);
    else if (a.dtype == FDB_DTYPE_F16) run<__half>(a, p);
    else run<__nv_bfloat16>(a, p);
}

// ---------------------------------------------------------------------------
// states
// ---------------------------------------------------------------------------
// Out of place: a block per run of a row.  In place: a block per 16 bytes x
// threads of all of a search's rows; a thread reads its bytes of every row before
// it writes any.
struct State {
    const unsigned char* src;
    unsigned char* dst;
    size_t src_stride, dst_stride, parts, src_part, dst_part, bytes;
};
__global__ void __launch_bounds__(256)
    move_kernel(const State t, const int64_t* __restrict__ parents, int beams, int width,
                int clear) {
    const size_t row = blockIdx.x / t.parts, part = blockIdx.x % t.parts;
    const size_t g = row / width;
    const int64_t from = parents[row];
    const bool none = from < 0 || from >= beams;
    if (none && !clear) return;
    const unsigned char* s = none ? nullptr : t.src + (g * beams + (size_t)from) * t.src_stride + part * t.src_part;
    unsigned char* d = t.dst + row * t.dst_stride + part * t.dst_part;
    for (size_t i = threadIdx.x; i < t.bytes; i += 256) d[i] = none ? 0 : s[i];
}
__global__ void __launch_bounds__(128)
    turn_kernel(const State t, const int64_t* __restrict__ parents, int beams) {
    extern __shared__ unsigned char held[];  // [beams][128]
    const size_t g = blockIdx.x / t.parts, part = blockIdx.x % t.parts;
    const size_t row0 = g * beams;
    for (size_t i = threadIdx.x; i < t.bytes; i += 128) {
        unsigned char* c = t.dst + row0 * t.dst_stride + part * t.dst_part + i;
        for (int b = 0; b < beams; ++b) {
            const int64_t from = parents[row0 + b];
            if (from >= 0 && from < beams) held[b * 128 + threadIdx.x] = c[from * t.dst_stride];
        }
        for (int b = 0; b < beams; ++b) {
            const int64_t from = parents[row0 + b];
            if (from >= 0 && from < beams) c[b * t.dst_stride] = held[b * 128 + threadIdx.x];
        }
    }
}
void reorder_run(const Ctx&, const fdb_beam_state* states, size_t count,
                 const fdb_reorder_opts& o) {
    const cudaStream_t s = static_cast<cudaStream_t>(o.stream);
    for (size_t i = 0; i < count; ++i) {
        const fdb_beam_state& a = states[i];
        if (a.bytes == 0 || a.parts == 0) continue;
        const State t{static_cast<const unsigned char*>(a.src), static_cast<unsigned char*>(a.dst),
                      a.src_stride, a.dst_stride, a.parts, a.src_part_stride, a.dst_part_stride,
                      a.bytes};
        if (a.src == a.dst)
            turn_kernel<<<(unsigned)(o.groups * a.parts), 128, o.beams * 128, s>>>(
                t, o.parents, (int)o.beams);
        else
            move_kernel<<<(unsigned)(o.groups * o.width * a.parts), 256, 0, s>>>(
                t, o.parents, (int)o.beams, (int)o.width, o.clear);
        FDB_LAUNCH_CHECK();
    }
}

}  // namespace beam
}  // namespace fdb
