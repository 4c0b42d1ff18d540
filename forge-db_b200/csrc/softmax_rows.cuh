// softmax_rows.cuh -- what operators on a softmax over rows share: conversions and
// passes over all scores that an operator ends in its own way.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fdb_internal.h"
#include "tc_ptx.cuh"

namespace fdb {
namespace sr {

constexpr double LOG2E = 1.4426950408889634074, LN2 = 0.69314718055994530942;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ---- pairs of f32 ----
__device__ __forceinline__ float lo_of(uint64_t v) {
    uint32_t a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
    return __uint_as_float(a);
}
__device__ __forceinline__ float hi_of(uint64_t v) {
    uint32_t a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
    return __uint_as_float(b);
}
__device__ __forceinline__ uint64_t packf(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(__float_as_uint(a)), "r"(__float_as_uint(b)));
    return d;
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
    return __bfloat162float(v);
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// Sums of q . x in 64 bits.  f32: products and sums in 64 bits (of a 64-bit copy
// of q); 16-bit types: the products are exact in f32, the sums in 64 bits.
template <typename T>
struct Exact {
    typedef float Q;
    double s = 0.0;
    __device__ __forceinline__ void add(float x, float q) { s += (double)__fmul_rn(x, q); }
    __device__ __forceinline__ double sum() const { return s; }
};
template <>
struct Exact<float> {
    typedef double Q;
    double s = 0.0;
    __device__ __forceinline__ void add(float x, double q) { s = fma((double)x, q, s); }
    __device__ __forceinline__ double sum() const { return s; }
};

// What a pass over the scores of queries [q0, q0 + nq) leaves: for part i and
// query q the triple part[i * nq + q] of fdb_logprobs' sums, in units of
// t = score * log2(e) as they were formed: f * rf for a score, with f = qf[q] (1 if
// null or 0) and rf the f32 nearest to scale * log2(e); `whole` puts right what
// the sums lost on average.  *err != 0: a wait ran out, the sums mean nothing.
struct Parts {
    const float4* part;
    int parts, q0, nq;
    const float* qf;
    double whole;
    const int* err;
};
// Ends the passes of forward_run in the place of fdb_logprobs' own end.
struct ForwardEnd {
    size_t queries;  // of one pass at most
    // Before a pass, if the call has filters of a query each (ld_allowed > 0):
    // those of its queries, the first one's first (`over`: see launch()).
    virtual const uint32_t* filters(size_t q0, size_t nq, bool over) = 0;
    virtual void finish(const Parts& p) = 0;
};
// Score gradients at given rows, in the place of what backward_run's formula
// gives there.
struct GivenRows {
    int k;                 // at most 256
    const int* row;        // [nq][k], each of a query once, < 0: none
    const float* g;        // [nq][k] dL / ds * scale
    const float* at_least; // [nq] a bound of their sizes over scale, >= 0
};

// What the caller of backward_run with given rows does before it: the exponents of the
// queries' bounds, and a cleared head of the workspace (weight null: neither).
struct BackwardHead {
    int* weight;      // [nq], weight_of(scale * at_least)
    uint32_t* clear;  // [words]
    int words;
};
constexpr int NO_WEIGHT = -10000;
__device__ __forceinline__ int weight_of(float bound) {
    return bound > 0.0f && bound <= 3.402823466e38f ? max(-110, ilogbf(bound)) : NO_WEIGHT;
}

size_t forward_bytes(const Ctx& c, const fdb_logprob_args& a, size_t pass_queries = 0);
void forward_run(Ctx& c, const fdb_logprob_args& a, ForwardEnd* end = nullptr);
size_t backward_bytes(const Ctx& c, const fdb_logprob_grad_args& a, const GivenRows* given = nullptr);
BackwardHead backward_head(const Ctx& c, const fdb_logprob_grad_args& a, const GivenRows& given);
void backward_run(Ctx& c, const fdb_logprob_grad_args& a, const GivenRows* given = nullptr);

// Raises a kernel's shared-memory limit once per device.  A kernel's limit is the
// process's, not the call's: `bytes` is the largest size that any call takes, as
// two threads may launch the same kernel at once.
template <typename K>
static void allow_smem(K* kernel, int device, size_t bytes, std::atomic<uint64_t>& done) {
    if (device < 64 && done.load(std::memory_order_acquire) >> device & 1u) return;
    FDB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    if (device < 64) done.fetch_or(1ull << device, std::memory_order_release);
}

// Kernels that follow one another in a call overlap: the next one's blocks take their
// places while the last one's end (some 1.5 us a launch).  Each of them waits, before it
// reads or writes anything that another one does, for all before it to be done: with
// one that did not, those after it would not know of those before.  What one of them
// left must not be read through a pointer that the compiler knows as the kernel's own
// (`const __restrict__`), as such a load may move ahead of the wait: see here().
__device__ __forceinline__ void wait_for_last() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
template <typename T>
__device__ __forceinline__ T* here(T* p) {
    asm volatile("" : "+l"(p)::"memory");
    return p;
}
// `over`: overlapping with the kernel before it, which is the same call's.
template <typename... P, typename... A>
static void launch(bool over, cudaStream_t s, void (*kernel)(P...), size_t blocks, int threads,
                   size_t smem, const A&... args) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t how{};
    how.gridDim = dim3((unsigned)blocks), how.blockDim = dim3((unsigned)threads);
    how.dynamicSmemBytes = smem, how.stream = s;
    how.attrs = &attr, how.numAttrs = over ? 1 : 0;
    FDB_CUDA(cudaLaunchKernelEx(&how, kernel, static_cast<P>(args)...));
}

inline size_t up(size_t v, size_t m) { return (v + m - 1) / m * m; }
// Hands out 256-byte aligned parts of the caller's workspace.
struct Carve {
    unsigned char* base;
    size_t at = 0;
    explicit Carve(void* b) : base(static_cast<unsigned char*>(b)) {}
    template <typename T>
    T* take(size_t count) {
        T* p = base ? reinterpret_cast<T*>(base + at) : nullptr;
        at += up(count * sizeof(T), 256);
        return p;
    }
};

}  // namespace sr
}  // namespace fdb
