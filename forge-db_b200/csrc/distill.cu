// distill.cu -- the loss of a teacher's best rows under a softmax over all rows,
// and its gradient.
//
//   P_e: the teacher's probabilities of the rows that it names, R = 1 - sum P
//   loss = sum_e P_e (log P_e - log p_e) [+ R (log R - log r)]
//   p_j = exp(s_j - lse),  r = sum of p over the rows that are not named
//   dL/ds_j = p_j - P_j at a named row,  p_j (1 - R / r) elsewhere
//
// The sums over all rows and the products are fdb_logprobs' (softmax_rows.cu).
// With `rest` the pass leaves the named rows out (by a filter for each query), as
// r = 1 - sum p loses all of its bits once the student is sure; their scores, in
// 64 bits, are joined to it.
#include <cmath>

#include "softmax_rows.cuh"

namespace fdb {
namespace distill {

using sr::Carve;
using sr::Exact;
using sr::LN2;
using sr::LOG2E;
using sr::to_f32;
using sr::up;

constexpr int MAXK = FDB_MAX_TEACHER;
constexpr size_t MASK_BYTES = (size_t)256 << 20;  // of one pass's filters

struct Teacher {
    const int64_t* ids;
    const float* z;
    size_t ld_ids, ld;  // ld: of z
    int k, n;
    double scale;
    int rest;
    const uint32_t* allowed;
    size_t ld_allowed;
};
__device__ __forceinline__ bool sees(const Teacher& t, int q, int64_t id) {
    return !t.allowed || (t.allowed[(size_t)q * t.ld_allowed + (size_t)(id >> 5)] >> (id & 31) & 1u);
}
// The row of an entry that may take part (whether an entry before it has the same
// id is left), else -1.
__device__ __forceinline__ int entry_row(const Teacher& t, int q, int e) {
    const int64_t id = t.ids[(size_t)q * t.ld_ids + e];
    if (id < 0 || id >= t.n || t.z[(size_t)q * t.ld + e] == -INFINITY || !sees(t, q, id)) return -1;
    return (int)id;
}

// ---- sums and maxima of C values over a block, the same bits in every thread ----
// (`part` [TH / 32][C] is the call's own: no barrier guards it from another use.)
template <int TH, int C, typename V, typename F>
__device__ __forceinline__ void block_all(V (&v)[C], V* part, F&& both) {
#pragma unroll
    for (int o = 16; o; o >>= 1)
#pragma unroll
        for (int c = 0; c < C; ++c) v[c] = both(v[c], __shfl_xor_sync(0xffffffffu, v[c], o));
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int c = 0; c < C; ++c) part[(threadIdx.x >> 5) * C + c] = v[c];
    __syncthreads();
#pragma unroll
    for (int c = 0; c < C; ++c) v[c] = part[c];
#pragma unroll
    for (int i = 1; i < TH / 32; ++i)
#pragma unroll
        for (int c = 0; c < C; ++c) v[c] = both(v[c], part[i * C + c]);
}
template <int TH, int C>
__device__ __forceinline__ void block_sums(double (&v)[C], double* part) {
    block_all<TH>(v, part, [](double a, double b) { return a + b; });
}
// (a NaN is passed over: the sums that follow carry it)
template <int TH, int C>
__device__ __forceinline__ void block_maxima(float (&v)[C], float* part) {
    block_all<TH>(v, part, [](float a, float b) { return fmaxf(a, b); });
}

// A query's entries in shared memory: the rows of those that take part, else -1.
template <int TH>
__device__ __forceinline__ void read_entries(const Teacher& t, int q, int* raw, int* row) {
    for (int e = threadIdx.x; e < t.k; e += TH) raw[e] = entry_row(t, q, e);
    __syncthreads();
    for (int e = threadIdx.x; e < t.k; e += TH) {
        int r = raw[e];
        for (int i = 0; r >= 0 && i < e; ++i)
            if (raw[i] == r) r = -1;
        row[e] = r;
    }
    __syncthreads();
}
// The teacher's part, from the largest logit zm of the entries that take part (-inf:
// there is none) and the sum of exp(scale (z - zm)): log P of an entry is
// scale z - norm, `left` is R.
struct Norm {
    double norm, left;
    bool any;
};
__device__ __forceinline__ Norm teacher_norm(const Teacher& t, float zm, double sum, bool any,
                                             bool others) {
    if (!any) return Norm{0.0, t.rest && others ? 1.0 : 0.0, false};
    Norm n{t.scale * (double)zm + log(sum), 0.0, true};
    if (t.rest && others && !(n.norm > 0.0)) {
        n.left = -expm1(n.norm);  // (NaN stays)
        n.norm = n.norm == n.norm ? 0.0 : NAN;
    }
    return n;
}
// exp(scale (z - zm)); of an infinite zm NaN, as it should be.
__device__ __forceinline__ double above(const Teacher& t, float z, float zm) {
    return exp(t.scale * ((double)z - (double)zm));
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
// Filters without the named rows, a block per query.  Bound by the latency of the words
// that a thread takes one after the other: 5 us for 1000 filters of 50001 rows, but of few
// queries over many rows with filters of their own more than the pass itself (one query of
// 1e7 rows: 1044 us where the pass takes 720; 22 without a filter).
__global__ void __launch_bounds__(128)
    filter_kernel(const Teacher t, int q0, uint32_t* __restrict__ out, size_t words) {
    const int q = q0 + (int)blockIdx.x;
    uint32_t* o = out + (size_t)blockIdx.x * words;
    const uint32_t* al = t.allowed ? t.allowed + (size_t)q * t.ld_allowed : nullptr;
    for (size_t w = threadIdx.x; w < words; w += 128) o[w] = al ? al[w] : 0xffffffffu;
    __syncthreads();
    for (int e = threadIdx.x; e < t.k; e += 128) {
        const int r = entry_row(t, q, e);
        if (r >= 0) atomicAnd(o + (r >> 5), ~(1u << (r & 31)));
    }
    sr::wait_for_last();  // (beside the packing of the rows)
}

struct LossArgs {
    Teacher t;
    sr::Parts parts;
    const void *q, *x;
    size_t ldq, ldx;
    int d;
    float scale;
    float *loss, *lse, *logprobs, *rest;
};
// Adds a vector's products with a query's to two sums, of the even and of the odd columns.
template <typename T, typename VT>
__device__ __forceinline__ void dot_vec(const VT& v, const typename Exact<T>::Q* q,
                                        Exact<T> (&sums)[2]) {
    constexpr int V = sizeof(VT) / sizeof(T);
    typedef typename Exact<T>::Q Q;
    const T* e = reinterpret_cast<const T*>(&v);
    Q y[V];
    // (16 bytes of the query at a time)
    constexpr int AT_ONCE = 16 / sizeof(Q) < V ? 16 / sizeof(Q) : V;
#pragma unroll
    for (int i = 0; i < V; i += AT_ONCE) {
        struct alignas(AT_ONCE * sizeof(Q)) Piece {
            Q y[AT_ONCE];
        };
        *reinterpret_cast<Piece*>(y + i) = *reinterpret_cast<const Piece*>(q + i);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) sums[i & 1].add(to_f32<T>(e[i]), y[i]);
}
// A lane's share of the products of ROWS rows with a query, by vectors of VT, in 64 bits: a
// sum in f32 is off by 2^-24 of its terms, which is much of a score that large terms leave of
// one another, and of the differences between named rows.  (f32 sums of four vectors: a call
// of 1000 lists of 64 rows of 768 bf16 86 us, so 90; 500 of 128 rows of 768 f32 51, so 61.)
// Two steps at a time for 16-byte vectors of 16-bit types (the first of those calls: 92 us
// with one), one for f32 (the second one: 74 us with two).
template <typename T, typename VT, int ROWS>
__device__ __forceinline__ void dot_rows(const T* const (&x)[ROWS], const typename Exact<T>::Q* q,
                                         int d, int sub, int lanes, double (&acc)[ROWS]) {
    constexpr int V = sizeof(VT) / sizeof(T), AHEAD = sizeof(T) == 4 ? 1 : V == 8 ? 2 : 4;
    Exact<T> sums[ROWS][2];
    int c = sub * V;
#pragma unroll AHEAD
    for (; c + V <= d; c += lanes * V) {
        VT v[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) v[r] = __ldg(reinterpret_cast<const VT*>(x[r] + c));
#pragma unroll
        for (int r = 0; r < ROWS; ++r) dot_vec<T, VT>(v[r], q + c, sums[r]);
    }
    // (the row's last, partial vector: one lane's)
    for (; c < d; ++c)
#pragma unroll
        for (int r = 0; r < ROWS; ++r) sums[r][0].add(to_f32<T>(x[r][c]), q[c]);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) acc[r] = sums[r][0].sum() + sums[r][1].sum();
}
// One block per query: the pass's sums joined, the named rows scored, the loss.  Gathers k
// rows a query, by vectors of what all rows are aligned to (a call of 2878 lists of 16 rows
// of 518 f16, aligned to 4 bytes: 65.5 us an element at a time, 64.9 by pairs).
template <typename T, int TH>
__global__ void __launch_bounds__(TH) loss_kernel(const LossArgs p) {
    extern __shared__ float4 q_raw[];
    typename Exact<T>::Q* qs = reinterpret_cast<typename Exact<T>::Q*>(q_raw);  // [dim]
    __shared__ int raw[MAXK], row[MAXK], list[MAXK];
    __shared__ double score[MAXK], sums[TH / 32][4], sums2[TH / 32];
    __shared__ float maxima[TH / 32][3];
    __shared__ int count;
    const int tid = threadIdx.x, ql = blockIdx.x, q = p.parts.q0 + ql;
    const T* qp = static_cast<const T*>(p.q) + (size_t)q * p.ldq;
    const T* xp = static_cast<const T*>(p.x);
    const float* z = p.t.z + (size_t)q * p.t.ld;
    if (tid == 0) count = 0;
    for (int c = tid; c < p.d; c += TH) qs[c] = to_f32<T>(qp[c]);
    read_entries<TH>(p.t, q, raw, row);
    for (int e = tid; e < p.t.k; e += TH)
        if (row[e] >= 0) list[atomicAdd(&count, 1)] = e;
    __syncthreads();

    // ---- the named rows' scores: 8 or 32 lanes a row, four rows at a time ----
    constexpr int ROWS = 4;
    const uintptr_t odd = reinterpret_cast<uintptr_t>(xp) | (p.ldx * sizeof(T));
    const int lanes = p.d * (int)sizeof(T) <= 512 ? 8 : 32, sub = tid & (lanes - 1);
    const int named = count, per = TH / lanes;
    for (int i = tid / lanes; i - tid / lanes < named; i += ROWS * per) {
        const T* x[ROWS];
        double acc[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
            x[r] = xp + (size_t)row[list[min(i + r * per, named - 1)]] * p.ldx;
        if ((odd & 15) == 0) dot_rows<T, uint4>(x, qs, p.d, sub, lanes, acc);
        else if ((odd & 7) == 0) dot_rows<T, uint2>(x, qs, p.d, sub, lanes, acc);
        else if (sizeof(T) == 4 || (odd & 3) == 0) dot_rows<T, unsigned>(x, qs, p.d, sub, lanes, acc);
        else if constexpr (sizeof(T) == 2) dot_rows<T, unsigned short>(x, qs, p.d, sub, lanes, acc);
#pragma unroll
        for (int o = 16; o; o >>= 1)
            if (o < lanes)
#pragma unroll
                for (int r = 0; r < ROWS; ++r) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
            if (sub == 0 && i + r * per < named) score[list[i + r * per]] = acc[r] * (double)p.scale;
    }
    // ---- the pass's sums (see finish_kernel): a thread's share ----
    // (until here nothing of the pass was read: blocks that found room were ahead of it)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const sr::Parts& ps = p.parts;
    float M = -INFINITY;
    double L = 0.0, A = 0.0;  // sums of 2^(t - M), and of those times t - M
    for (int i = tid; i < ps.parts; i += TH) {
        const float4 v = ps.part[(size_t)i * ps.nq + ql];
        if (v.y == 0.0f && v.z == 0.0f) continue;
        if (v.x > M) {
            if (L != 0.0) {
                const double e = (double)sr::ex2(M - v.x);
                A = (A + ((double)M - (double)v.x) * L) * e;
                L *= e;
            }
            M = v.x;
        }
        const float e = v.x == M ? 1.0f : sr::ex2(v.x - M);
        L += v.z == v.z ? (double)(v.y * e) : NAN;
        A += ((double)v.z + ((double)v.x - (double)M) * (double)v.y) * (double)e;
    }
    __syncthreads();

    // ---- maxima: of the pass's references, of the logits, of the named scores ----
    float mx[3] = {M, -INFINITY, -INFINITY};
    for (int e = tid; e < p.t.k; e += TH)
        if (row[e] >= 0) mx[1] = fmaxf(mx[1], z[e]), mx[2] = fmaxf(mx[2], (float)score[e]);
    block_maxima<TH>(mx, &maxima[0][0]);
    const float zm = mx[1];
    const double tm = mx[2];
    // ---- sums relative to them ----
    const double to_all = M == mx[0] || L == 0.0 ? 1.0 : (double)sr::ex2(M - mx[0]);
    double sum[4] = {L == 0.0 ? 0.0 : L * to_all, 0.0, 0.0,
                     L == 0.0 ? 0.0 : (A + ((double)M - (double)mx[0]) * L) * to_all};
    for (int e = tid; e < p.t.k; e += TH)
        if (row[e] >= 0) {
            sum[1] += above(p.t, z[e], zm);
            sum[2] += fabs(score[e]) < INFINITY ? exp(score[e] - tm) : NAN;
        }
    block_sums<TH>(sum, &sums[0][0]);
    L = sum[0], A = sum[3];
    const bool bad = !(L == L) || *ps.err != 0;
    float f = 1.0f;
    if (ps.qf) f = ps.qf[ql] == 0.0f ? 1.0f : ps.qf[ql];
    const double unit = (double)p.scale * LOG2E;
    const float rf = f * (float)unit;
    const bool others = !p.t.rest || L > 0.0;
    // Each t was formed with rf, rounded to f32, from a sum that was cut: short of itself by
    // a share `off` on average.  A share of every score moves the lse by that share of their
    // mean under the softmax, A / L above the reference.  (Of the reference itself it is too
    // much by what that lies above the mean: log r off by 1.8e-6 of its norm, 3.6e-7 so, at
    // 60 x 48639 x 981 f16.)
    const double off = (double)f * unit / (double)rf * ps.whole - 1.0;
    const double rest_lse = bad       ? NAN
                            : L > 0.0 ? LN2 * ((double)mx[0] + off * ((double)mx[0] + A / L)) + log(L)
                                      : -INFINITY;
    double lse = rest_lse;
    if (p.t.rest && named > 0) {  // (the named rows were left out)
        const double t = fmax(tm, rest_lse);
        lse = t + log(sum[2] * exp(tm - t) + exp(rest_lse - t));
    }
    const Norm nm = teacher_norm(p.t, zm, sum[1], named > 0, others);
    double loss[1] = {0.0};
    for (int e = tid; e < p.t.k; e += TH) {
        const double lp = row[e] >= 0 ? score[e] - lse : 0.0;
        if (row[e] >= 0) {
            const double lt = p.t.scale * (double)z[e] - nm.norm, w = exp(lt);
            if (!(w == 0.0)) loss[0] += w * (lt - lp);
        }
        if (p.logprobs) p.logprobs[(size_t)q * p.t.k + e] = (float)(lse == lse ? lp : NAN);
    }
    block_sums<TH>(loss, sums2);
    if (tid != 0) return;
    const double rest = lse == -INFINITY || rest_lse == -INFINITY ? -INFINITY : rest_lse - lse;
    if (p.t.rest && nm.any && nm.left > 0.0) loss[0] += nm.left * (log(nm.left) - rest);
    // (a divergence: what lies below 0 is the scores' and the lse's rounding, which come
    // from different sums; a NaN stays)
    if (loss[0] < 0.0) loss[0] = 0.0;
    // (not finite: a query or a row that counts, or a named row with a weight of 0)
    if (!(lse == lse)) loss[0] = NAN;
    if (p.loss) p.loss[q] = (float)loss[0];
    if (p.lse) p.lse[q] = (float)lse;
    if (p.rest) p.rest[q] = (float)rest;
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
struct CoefArgs {
    Teacher t;
    double scale;
    const float *lse, *logprobs, *rest, *d_loss;
    int* row;                         // [nq][k], see GivenRows
    float *g, *at_least, *ref, *c;    // G elsewhere = scale c exp(s - ref)
    sr::BackwardHead head;
};
// One block per query: what the score gradients are formed with.  A chain of short steps;
// a warp where a list is short enough, as a barrier of one warp costs nothing (2048 lists
// of 32: 12.0 us with 128 threads).
template <int TH>
__global__ void __launch_bounds__(TH) grad_kernel(const CoefArgs p) {
    __shared__ int raw[MAXK], row[MAXK];
    __shared__ double sums[TH / 32];
    __shared__ float maxima[TH / 32];
    sr::wait_for_last();
    const int tid = threadIdx.x, q = blockIdx.x;
    if (q == 0)
        for (int i = tid; i < p.head.words; i += TH) p.head.clear[i] = 0u;
    const float lse = p.lse[q], rest = p.t.rest ? p.rest[q] : 0.0f, up = p.d_loss[q];
    read_entries<TH>(p.t, q, raw, row);
    const bool others = rest > -INFINITY || !(rest == rest);
    const float* z = p.t.z + (size_t)q * p.t.ld;
    float zm[1] = {-INFINITY};
    bool mine = false;
    for (int e = tid; e < p.t.k; e += TH)
        if (row[e] >= 0) zm[0] = fmaxf(zm[0], z[e]), mine = true;
    const bool any = __syncthreads_or(mine);
    block_maxima<TH>(zm, maxima);
    double sum[1] = {0.0};
    for (int e = tid; e < p.t.k; e += TH)
        if (row[e] >= 0) sum[0] += above(p.t, z[e], zm[0]);
    block_sums<TH>(sum, sums);
    const Norm nm = teacher_norm(p.t, zm[0], sum[0], any, others);
    const bool live = nm.any && lse != -INFINITY;
    const double u = live ? (double)up : 0.0;
    const size_t at = (size_t)q * p.t.k;
    for (int e = tid; e < p.t.k; e += TH) {
        p.row[at + e] = live ? row[e] : -1;
        if (row[e] < 0) continue;
        const double w = exp(p.t.scale * (double)z[e] - nm.norm);
        p.g[at + e] = (float)(p.scale * u * (exp((double)p.logprobs[at + e]) - w));
    }
    if (tid != 0) return;
    p.at_least[q] = (float)fabs(u);
    if (p.head.weight) p.head.weight[q] = sr::weight_of((float)(p.scale * fabs(u)));
    p.ref[q] = others ? (float)((double)lse + (double)rest) : lse;
    double c = u * ((p.t.rest ? exp((double)rest) : 1.0) - nm.left);
    if (live && !(nm.norm == nm.norm)) c = NAN;
    p.c[q] = live ? (float)c : 0.0f;
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
template <typename A>
static Teacher teacher_of(const A& a) {
    Teacher t{};
    t.ids = a.teacher_ids, t.z = a.teacher_logits;
    t.ld_ids = a.ld_ids, t.ld = a.ld_logits;
    t.k = (int)a.k, t.n = (int)a.n;
    t.scale = a.teacher_scale, t.rest = a.rest != 0;
    t.allowed = a.allowed, t.ld_allowed = a.allowed ? a.ld_allowed : 0;
    return t;
}
template <typename H, typename A>
static H head_of(const A& a) {
    H h{};
    h.dtype = a.dtype;
    h.queries = a.queries, h.nq = a.nq, h.ld_queries = a.ld_queries;
    h.rows = a.rows, h.n = a.n, h.ld_rows = a.ld_rows;
    h.dim = a.dim, h.scale = a.scale;
    h.allowed = a.allowed, h.ld_allowed = a.ld_allowed;
    h.workspace = a.workspace, h.stream = a.stream;
    return h;
}

struct Plan {
    fdb_logprob_args head;
    size_t words, queries;  // of a filter, of a pass (0: any)
    uint32_t* filters;
    size_t bytes;
};
static Plan plan_forward(const Ctx& c, const fdb_distill_args& a) {
    Plan p{};
    p.head = head_of<fdb_logprob_args>(a);
    p.words = (a.n + 31) / 32;
    if (a.rest) {
        // (the filters are the pass's: the address only has to say that there are some)
        p.queries = std::min(a.nq, std::max<size_t>(256, MASK_BYTES / (p.words * 4) / 256 * 256));
        p.head.allowed = reinterpret_cast<const uint32_t*>(256);
        p.head.ld_allowed = p.words;
    }
    p.bytes = up(sr::forward_bytes(c, p.head, p.queries), 256);
    if (a.rest) {
        p.filters = reinterpret_cast<uint32_t*>(static_cast<unsigned char*>(a.workspace) + p.bytes);
        p.bytes += up(p.queries * p.words * 4, 256);
    }
    return p;
}
size_t forward_bytes(const Ctx& c, const fdb_distill_args& a) { return plan_forward(c, a).bytes; }

template <typename T, int TH>
static void launch_loss(cudaStream_t s, int device, const LossArgs& p) {
    typedef typename Exact<T>::Q Q;
    const size_t smem = up((size_t)p.d * sizeof(Q), 16);
    if (smem > 32768) {  // (with the static part, over what needs no permission)
        static std::atomic<uint64_t> done{0};
        sr::allow_smem(loss_kernel<T, TH>, device, FDB_MAX_SOFTMAX_DIM * sizeof(Q), done);
    }
    sr::launch(true, s, loss_kernel<T, TH>, p.parts.nq, TH, smem, p);
}
template <typename T>
static void launch_loss(cudaStream_t s, int device, int sms, const LossArgs& p) {
    // Few queries: more threads share the rows of one.  Many: as few as leave all blocks
    // resident at once, where a chain of short steps is what a block waits for (2048 lists
    // of 32 rows of 768 bf16: 37 us with 128 threads, 29 with 64).
    if (p.parts.nq <= 2 * sms) launch_loss<T, 512>(s, device, p);
    else if (p.parts.nq <= 8 * sms) launch_loss<T, 128>(s, device, p);
    else launch_loss<T, 64>(s, device, p);
}

struct End : sr::ForwardEnd {
    const Ctx& c;
    const fdb_distill_args& a;
    const Plan& plan;
    cudaStream_t s;
    End(const Ctx& c_, const fdb_distill_args& a_, const Plan& p)
        : c(c_), a(a_), plan(p), s(static_cast<cudaStream_t>(a_.stream)) {
        queries = p.queries;
    }
    const uint32_t* filters(size_t q0, size_t nq, bool over) override {
        const Teacher t = teacher_of(a);
        if (!a.rest) return a.allowed + q0 * a.ld_allowed;
        sr::launch(over, s, filter_kernel, nq, 128, 0, t, (int)q0, plan.filters, plan.words);
        return plan.filters;
    }
    void finish(const sr::Parts& parts) override {
        LossArgs p{};
        p.t = teacher_of(a);
        p.parts = parts;
        p.q = a.queries, p.ldq = a.ld_queries;
        p.x = a.rows, p.ldx = a.ld_rows;
        p.d = (int)a.dim, p.scale = a.scale;
        p.loss = a.loss, p.lse = a.lse, p.logprobs = a.logprobs;
        p.rest = a.rest ? a.rest_logprob : nullptr;
        if (a.dtype == FDB_DTYPE_F32) launch_loss<float>(s, c.device, c.sm_count, p);
        else if (a.dtype == FDB_DTYPE_F16) launch_loss<__half>(s, c.device, c.sm_count, p);
        else launch_loss<__nv_bfloat16>(s, c.device, c.sm_count, p);
    }
};
void forward_run(Ctx& c, const fdb_distill_args& a) {
    const Plan p = plan_forward(c, a);
    End end(c, a, p);
    sr::forward_run(c, p.head, &end);
}

struct BackwardPlan {
    fdb_logprob_grad_args head;
    sr::GivenRows given;
    CoefArgs k;
    size_t bytes;
};
static BackwardPlan plan_backward(const Ctx& c, const fdb_distill_grad_args& a) {
    BackwardPlan p{};
    p.head = head_of<fdb_logprob_grad_args>(a);
    p.head.d_queries = a.d_queries, p.head.ld_d_queries = a.ld_d_queries;
    p.head.d_rows = a.d_rows, p.head.ld_d_rows = a.ld_d_rows;
    p.given.k = (int)a.k;
    const size_t first = up(sr::backward_bytes(c, p.head, &p.given), 256);
    Carve ws(a.workspace ? static_cast<unsigned char*>(a.workspace) + first : nullptr);
    CoefArgs& k = p.k;
    k.row = ws.take<int>(a.nq * a.k);
    k.g = ws.take<float>(a.nq * a.k);
    k.at_least = ws.take<float>(a.nq);
    k.ref = ws.take<float>(a.nq);
    k.c = ws.take<float>(a.nq);
    p.given.row = k.row, p.given.g = k.g, p.given.at_least = k.at_least;
    p.head.lse = k.ref, p.head.d_lse = k.c;
    p.bytes = first + ws.at;
    return p;
}
size_t backward_bytes(const Ctx& c, const fdb_distill_grad_args& a) {
    fdb_distill_grad_args b = a;
    b.workspace = nullptr;
    return plan_backward(c, b).bytes;
}
void backward_run(Ctx& c, const fdb_distill_grad_args& a) {
    BackwardPlan p = plan_backward(c, a);
    CoefArgs& k = p.k;
    k.t = teacher_of(a);
    k.scale = a.scale;
    k.lse = a.lse, k.logprobs = a.logprobs, k.rest = a.rest_logprob, k.d_loss = a.d_loss;
    k.head = sr::backward_head(c, p.head, p.given);
    const cudaStream_t s = static_cast<cudaStream_t>(a.stream);
    if (a.k <= 64) grad_kernel<32><<<(unsigned)a.nq, 32, 0, s>>>(k);
    else grad_kernel<128><<<(unsigned)a.nq, 128, 0, s>>>(k);
    FDB_LAUNCH_CHECK();
    sr::backward_run(c, p.head, &p.given);
}

}  // namespace distill
}  // namespace fdb
