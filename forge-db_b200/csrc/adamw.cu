// adamw.cu -- one AdamW step over many tensors, moments in f32 or 8 bits.
//
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Every operation is rounded in f32 by itself and in this order.  8-bit
// moments (blocks of 256 elements, s = the block's largest |m| or v):
//   m = s c |c| / 127^2, c in [-127, 127];   v = s c^4 / 255^4, c in [0, 255]
// so that small values keep a relative step (the fourth power because the
// update divides by sqrt(v)).  A value between two codes goes up with a
// probability equal to its distance from the lower one: the step changes v by
// a thousandth, far less than a code, and rounding to nearest would never
// move it.  The draw is a hash of (seed, step, tensor, element).  v > 0 keeps
// a code of at least 1: a zero under a moment that is not zero would make the
// update m / eps.  v is a square, so a block whose largest v is small (gradients
// below about 1e-12) is held and read 2^64 larger, down to 2^-112; below that
// (gradients below about 1e-15) its v is held as zeros, and its m with it.
//
// Bound by memory with f32 moments: f32 p, g, m, v move 28 bytes an element
// (131072 x 768: 419 us, 6.7 TB/s).  bf16 p, g with 8-bit moments move 10, and
// 147 instructions an element take longer than that (40 M elements: 203 us).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "fdb_internal.h"

namespace fdb {
namespace adamw {

constexpr int TENSORS = 96;      // tensors a launch takes (their table is a kernel argument)
constexpr int THREADS = 256;
constexpr int CHUNK = 8192;      // elements a block works through
constexpr int SMALL_CHUNK = 2048;  // ... when there are too few for every multiprocessor
constexpr int BLOCK8 = FDB_ADAMW_BLOCK;
// A block whose largest |m| is below LEAST, or largest v below LEAST_V, holds zeros;
// one whose largest v is below LEAST is worked on UP times larger (255^4 / v has to
// stay in range, and v / 255^4 out of f32's subnormal numbers).
constexpr float LEAST = 0x1p-90f, LEAST_V = 0x1p-112f, UP = 0x1p64f;
constexpr float M_CODES = 16129.0f, V_CODES = 4228250625.0f;  // 127^2, 255^4

struct Entry {
    void* p;
    const void* g;
    void *m, *v;
    float *ms, *vs;
    size_t n;
    unsigned first;    // first block of the launch that works on it
    unsigned ordinal;  // number of the tensor in the call
    unsigned wide;     // every pointer is aligned for whole-vector accesses
};
struct Table {
    Entry e[TENSORS];
    int count;
};
struct Hyper {
    double lr, b1, b2, wd;
    float eps, grad_scale;
    int64_t step;
    uint32_t seed;
    const float *d_lr, *d_grad_scale;
    const int64_t* d_step;
    int on_device;  // some of them are read when the kernel runs
};
// The constants of a step, each rounded once from 64 bits.
struct Consts {
    float b1, c1, b2, c2, keep, rate, root, eps, gs;
    uint32_t salt;
};
__host__ __device__ inline Consts consts_of(const Hyper& h, double lr, int64_t t, float gs) {
    Consts c;
    c.b1 = (float)h.b1, c.c1 = (float)(1.0 - h.b1);
    c.b2 = (float)h.b2, c.c2 = (float)(1.0 - h.b2);
    c.keep = (float)(1.0 - lr * h.wd);
    c.rate = (float)(lr / (1.0 - pow(h.b1, (double)t)));
    c.root = (float)(1.0 / sqrt(1.0 - pow(h.b2, (double)t)));
    c.eps = h.eps;
    c.gs = gs;
    c.salt = h.seed + ((uint32_t)t << 16);
    return c;
}
// The constants of the step in a block: the host's, or from the device values.
__device__ __forceinline__ Consts step_consts(const Hyper& h, const Consts& given, Consts* shared) {
    if (!h.on_device) return given;
    if (threadIdx.x == 0)
        *shared = consts_of(h, h.d_lr ? (double)*h.d_lr : h.lr, h.d_step ? *h.d_step : h.step,
                            h.d_grad_scale ? __fmul_rn(h.grad_scale, *h.d_grad_scale)
                                           : h.grad_scale);
    __syncthreads();
    return *shared;
}

template <typename T>
__device__ __forceinline__ float get(T v);
template <>
__device__ __forceinline__ float get<float>(float v) { return v; }
template <>
__device__ __forceinline__ float get<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float get<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T put(float v);
template <>
__device__ __forceinline__ float put<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 put<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half put<__half>(float v) { return __float2half_rn(v); }

// N consecutive elements (N * sizeof(T) a power of two, aligned to it up to 16).
template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Vec {
    T e[N];
};

__device__ __forceinline__ void moments(const Consts& c, float b2, float g, float& m, float& v) {
    m = __fadd_rn(__fmul_rn(m, c.b1), __fmul_rn(g, c.c1));
    v = __fadd_rn(__fmul_rn(v, b2), __fmul_rn(__fmul_rn(g, g), c.c2));
}
__device__ __forceinline__ float stepped(const Consts& c, float p, float m, float v) {
    const float den = __fadd_rn(__fmul_rn(__fsqrt_rn(v), c.root), c.eps);
    return __fsub_rn(__fmul_rn(p, c.keep), __fmul_rn(__fdiv_rn(m, den), c.rate));
}

// The published 32-bit mixer lowbias32: its shifts and constants.
__device__ __forceinline__ uint32_t mix(uint32_t h) {
    h = (h ^ (h >> 16)) * 0x7FEB352Du;
    h = (h ^ (h >> 15)) * 0x846CA68Bu;
    return h ^ (h >> 16);
}
__device__ __forceinline__ float unit(uint32_t h) { return (float)(h >> 8) * 0x1p-24f; }

// Conversions between small integers and floats go by adding 2^23, whose low
// mantissa bits then are the integer: a quarter of the cycles of the conversion
// instructions, of which a code would need ten.
__device__ __forceinline__ float fast_sqrt(float y) {
    float r;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
    return r;
}
__device__ __forceinline__ float nearest(float r) {  // 0 <= r < 2^22
    return __fsub_rn(__fadd_rn(r, 8388608.0f), 8388608.0f);
}
__device__ __forceinline__ float below(float r, float n) { return r < n ? n - 1.0f : n; }
// Byte `i` of w as a float, less `off`.
__device__ __forceinline__ float byte_float(uint32_t w, int i, float off) {
    return __fsub_rn(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7540 + i)), 8388608.0f + off);
}
// Whole numbers in [-128, 255] as the low bytes of four words, and these as one.
__device__ __forceinline__ uint32_t low_byte(float k) {
    return __float_as_uint(__fadd_rn(k, 12582912.0f));
}
__device__ __forceinline__ uint32_t pack_bytes(const uint32_t* w) {
    return __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
}
// The larger of the two, NaN if one is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// The codes of y = |m| (127^2 / scale) and z = v (255^4 / scale): the root's
// floor k, or k + 1 if u < (y - k^p) / ((k + 1)^p - k^p), p = 2 or 4.
__device__ __forceinline__ float code_m_exact(float y, float u) {
    const float r = __fsqrt_rn(y), k = below(r, nearest(r)), lo = __fmul_rn(k, k);
    const float k1 = __fadd_rn(k, 1.0f), hi = __fmul_rn(k1, k1);
    return u < __fdiv_rn(__fsub_rn(y, lo), __fsub_rn(hi, lo)) ? k1 : k;
}
__device__ __forceinline__ float code_v_exact(float z, float u) {
    const float r = __fsqrt_rn(__fsqrt_rn(z)), k = below(r, nearest(r));
    const float k1 = __fadd_rn(k, 1.0f), l = __fmul_rn(k, k), h = __fmul_rn(k1, k1);
    const float lo = __fmul_rn(l, l), hi = __fmul_rn(h, h);
    return u < __fdiv_rn(__fsub_rn(z, lo), __fsub_rn(hi, lo)) ? k1 : k;
}
// The same from approximate roots and without the division, and whether that
// may differ (one branch then leads to the exact ones; a warp takes it for one
// element in fifty).  u is compared with the quotient by the sign of u w - a,
// certain where that is more than the roundings of both sides.  The roots are
// off by less than 2^-22 of themselves, so a floor is wrong only if the root
// is that close to a whole number n <= 255: the quotient is then within 2^-13
// of 1 from n - 1 and of 0 from n, and both give n unless u is as close to
// either.  (Testing the root instead would find every block's largest element.)
__device__ __forceinline__ bool extreme(float u) {
    return fabsf(__fsub_rn(u, 0.5f)) >= 0.5f - 0x1p-13f;
}
__device__ __forceinline__ float code_m(float y, float u, bool& unsure) {
    const float r = fast_sqrt(y), k = below(r, nearest(r));
    // (k^2 and 2 k + 1 are exact, so both are rounded as in the exact form)
    const float a = __fmaf_rn(-k, k, y), w = __fmaf_rn(2.0f, k, 1.0f), t = __fmaf_rn(u, w, -a);
    unsure = extreme(u) || fabsf(t) <= w * 0x1p-21f;
    return t < 0.0f ? __fadd_rn(k, 1.0f) : k;
}
__device__ __forceinline__ float code_v(float z, float u, bool& unsure) {
    const float r = fast_sqrt(fast_sqrt(z)), k = below(r, nearest(r));
    const float k1 = __fadd_rn(k, 1.0f), l = __fmul_rn(k, k), h = __fmul_rn(k1, k1);
    const float lo = __fmul_rn(l, l), w = __fsub_rn(__fmul_rn(h, h), lo);
    const float t = __fmaf_rn(u, w, -__fsub_rn(z, lo));
    unsure = extreme(u) || fabsf(t) <= w * 0x1p-21f;
    return t < 0.0f ? k1 : k;
}

__device__ __forceinline__ const Entry& entry_of(const Table& t, unsigned block) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.e[mid].first <= block) lo = mid;
        else hi = mid - 1;
    }
    return t.e[lo];
}

template <typename P, typename G>
__global__ void __launch_bounds__(THREADS)
    step32_kernel(const __grid_constant__ Table t, const __grid_constant__ Hyper h,
                  const __grid_constant__ Consts given, int chunk) {
    __shared__ Consts sc;
    const Consts c = step_consts(h, given, &sc);
    const Entry& e = entry_of(t, blockIdx.x);
    P* p = static_cast<P*>(e.p);
    const G* g = static_cast<const G*>(e.g);
    float *m = static_cast<float*>(e.m), *v = static_cast<float*>(e.v);
    const size_t n = e.n, i0 = (size_t)(blockIdx.x - e.first) * chunk;
    const size_t i1 = min(n, i0 + chunk);
    constexpr int N = 4, U = 2;
    if (e.wide && (i1 - i0) % (THREADS * N * U) == 0) {
#pragma unroll 1
        for (int r = 0; r < (int)(i1 - i0) / (THREADS * N * U); ++r) {
            Vec<P, N> pv[U];
            Vec<G, N> gv[U];
            Vec<float, N> mv[U], vv[U];
            const size_t b = i0 + (size_t)r * THREADS * N * U + (size_t)threadIdx.x * N;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const size_t i = b + (size_t)u * THREADS * N;
                gv[u] = *reinterpret_cast<const Vec<G, N>*>(g + i);
                mv[u] = *reinterpret_cast<const Vec<float, N>*>(m + i);
                vv[u] = *reinterpret_cast<const Vec<float, N>*>(v + i);
                pv[u] = *reinterpret_cast<const Vec<P, N>*>(p + i);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const size_t i = b + (size_t)u * THREADS * N;
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    moments(c, c.b2, __fmul_rn(get<G>(gv[u].e[j]), c.gs), mv[u].e[j], vv[u].e[j]);
                    pv[u].e[j] =
                        put<P>(stepped(c, get<P>(pv[u].e[j]), mv[u].e[j], vv[u].e[j]));
                }
                *reinterpret_cast<Vec<P, N>*>(p + i) = pv[u];
                *reinterpret_cast<Vec<float, N>*>(m + i) = mv[u];
                *reinterpret_cast<Vec<float, N>*>(v + i) = vv[u];
            }
        }
        return;
    }
    for (size_t i = i0 + threadIdx.x; i < i1; i += THREADS) {
        float mi = m[i], vi = v[i];
        moments(c, c.b2, __fmul_rn(get<G>(g[i]), c.gs), mi, vi);
        p[i] = put<P>(stepped(c, get<P>(p[i]), mi, vi));
        m[i] = mi;
        v[i] = vi;
    }
}

// One warp per block of 256 elements, 8 consecutive ones a lane.
template <typename P, typename G>
__global__ void __launch_bounds__(THREADS)
    step8_kernel(const __grid_constant__ Table t, const __grid_constant__ Hyper h,
                  const __grid_constant__ Consts given, int chunk) {
    __shared__ Consts sc;
    const Consts c = step_consts(h, given, &sc);
    const Entry& e = entry_of(t, blockIdx.x);
    P* p = static_cast<P*>(e.p);
    const G* g = static_cast<const G*>(e.g);
    int8_t* m8 = static_cast<int8_t*>(e.m);
    uint8_t* v8 = static_cast<uint8_t*>(e.v);
    const size_t n = e.n, i0 = (size_t)(blockIdx.x - e.first) * chunk;
    const size_t i1 = min(n, i0 + chunk);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t salt = mix(c.salt + e.ordinal);
    constexpr float KM = (float)(1.0 / 16129.0), KV = (float)(1.0 / 4228250625.0);
    for (size_t b0 = i0 + (size_t)warp * BLOCK8; b0 < i1; b0 += (THREADS / 32) * BLOCK8) {
        const size_t i = b0 + (size_t)lane * 8, blk = b0 / BLOCK8;
        Vec<P, 8> pv;
        Vec<G, 8> gv;
        uint2 mc = make_uint2(0, 0), vc = make_uint2(0, 0);  // eight codes each
        const bool wide = e.wide && b0 + BLOCK8 <= i1;
        if (wide) {
            gv = *reinterpret_cast<const Vec<G, 8>*>(g + i);
            pv = *reinterpret_cast<const Vec<P, 8>*>(p + i);
            mc = *reinterpret_cast<const uint2*>(m8 + i);
            vc = *reinterpret_cast<const uint2*>(v8 + i);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool in = i + j < i1;
                gv.e[j] = in ? g[i + j] : put<G>(0.0f);
                pv.e[j] = in ? p[i + j] : put<P>(0.0f);
                const uint32_t a = in ? (uint8_t)m8[i + j] : 0u, b = in ? v8[i + j] : 0u;
                (j < 4 ? mc.x : mc.y) |= a << (8 * (j & 3));
                (j < 4 ? vc.x : vc.y) |= b << (8 * (j & 3));
            }
        }
        const float ks = __fmul_rn(e.ms[blk], KM), s0 = e.vs[blk];
        const float kv = __fmul_rn(s0 < LEAST ? __fmul_rn(s0, UP) : s0, KV);
        const float b2 = s0 < LEAST ? __fmul_rn(c.b2, 1.0f / UP) : c.b2;  // (and back)
        float m[8], v[8], sm = 0.0f, sv = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // (signed codes as c + 128)
            const float a = byte_float((j < 4 ? mc.x : mc.y) ^ 0x80808080u, j & 3, 128.0f);
            const float r = byte_float(j < 4 ? vc.x : vc.y, j & 3, 0.0f);
            m[j] = __fmul_rn(__fmul_rn(a, fabsf(a)), ks);
            const float r2 = __fmul_rn(r, r);
            v[j] = __fmul_rn(__fmul_rn(r2, r2), kv);
            moments(c, b2, __fmul_rn(get<G>(gv.e[j]), c.gs), m[j], v[j]);
            pv.e[j] = put<P>(stepped(c, get<P>(pv.e[j]), m[j], v[j]));
            // (past the tensor's end: zeros.  A NaN makes the block's scale NaN: the
            // block reads as NaN from then on)
            sm = max_nan(sm, fabsf(m[j]));
            sv = max_nan(sv, v[j]);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            sm = max_nan(sm, __shfl_xor_sync(0xffffffffu, sm, o));
            sv = max_nan(sv, __shfl_xor_sync(0xffffffffu, sv, o));
        }
        if (sv > 0.0f && sv < LEAST_V) sm = 0.0f;
        const float km = sm > LEAST ? __fdiv_rn(M_CODES, sm) : 0.0f;
        float kw = sv > LEAST ? __fdiv_rn(V_CODES, sv) : 0.0f;
        if (sv >= LEAST_V && sv <= LEAST) {
            kw = __fdiv_rn(V_CODES, __fmul_rn(sv, UP));
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], UP);
        }
        // (i is a multiple of 8: the eight numbers differ in their last bits)
        const uint32_t at =
            (uint32_t)i ^ salt ^ ((uint32_t)((uint64_t)i >> 32) * 0x9E3779B1u);
        uint32_t mb[8], vb[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t hh = mix(at ^ (uint32_t)j);
            const float um = unit(hh), uv = unit(mix(hh ^ 0x5BD1E995u));
            const float y = __fmul_rn(fabsf(m[j]), km), z = __fmul_rn(v[j], kw);
            bool unsure_m, unsure_v;
            float k = code_m(y, um, unsure_m), l = code_v(z, uv, unsure_v);
            if (unsure_m || unsure_v) k = code_m_exact(y, um), l = code_v_exact(z, uv);
            mb[j] = low_byte(copysignf(fminf(k, 127.0f), m[j]));
            vb[j] = low_byte(z > 0.0f ? fmaxf(fminf(l, 255.0f), 1.0f) : 0.0f);
        }
        mc = make_uint2(pack_bytes(mb), pack_bytes(mb + 4));
        vc = make_uint2(pack_bytes(vb), pack_bytes(vb + 4));
        if (wide) {
            *reinterpret_cast<Vec<P, 8>*>(p + i) = pv;
            *reinterpret_cast<uint2*>(m8 + i) = mc;
            *reinterpret_cast<uint2*>(v8 + i) = vc;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + j < i1) {
                    p[i + j] = pv.e[j];
                    m8[i + j] = (int8_t)((j < 4 ? mc.x : mc.y) >> (8 * (j & 3)));
                    v8[i + j] = (uint8_t)((j < 4 ? vc.x : vc.y) >> (8 * (j & 3)));
                }
        }
        if (lane == 0) {
            e.ms[blk] = sm < LEAST ? 0.0f : sm;
            e.vs[blk] = sv < LEAST_V ? 0.0f : sv;
        }
    }
}

// The values that 8-bit moments stand for.
__global__ void __launch_bounds__(THREADS)
    values_kernel(const int8_t* __restrict__ m, const float* __restrict__ ms,
                  const uint8_t* __restrict__ v, const float* __restrict__ vs, size_t n,
                  float* __restrict__ om, float* __restrict__ ov, int wide) {
    constexpr float KM = (float)(1.0 / 16129.0), KV = (float)(1.0 / 4228250625.0);
    const size_t step = (size_t)gridDim.x * THREADS * 4;
    for (size_t i = ((size_t)blockIdx.x * THREADS + threadIdx.x) * 4; i < n; i += step) {
        const float ks = __fmul_rn(ms[i / BLOCK8], KM), s0 = vs[i / BLOCK8];
        const float kv = __fmul_rn(s0 < LEAST ? __fmul_rn(s0, UP) : s0, KV);
        const float down = s0 < LEAST ? 1.0f / UP : 1.0f;
        const bool whole = wide && i + 4 <= n;
        Vec<int8_t, 4> mc;
        Vec<uint8_t, 4> vc;
        if (whole) {
            mc = *reinterpret_cast<const Vec<int8_t, 4>*>(m + i);
            vc = *reinterpret_cast<const Vec<uint8_t, 4>*>(v + i);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                mc.e[j] = i + j < n ? m[i + j] : (int8_t)0;
                vc.e[j] = i + j < n ? v[i + j] : (uint8_t)0;
            }
        }
        Vec<float, 4> a, b;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float x = (float)mc.e[j], r = (float)vc.e[j], r2 = __fmul_rn(r, r);
            a.e[j] = __fmul_rn(__fmul_rn(x, fabsf(x)), ks);
            b.e[j] = __fmul_rn(__fmul_rn(__fmul_rn(r2, r2), kv), down);
        }
        if (whole) {
            *reinterpret_cast<Vec<float, 4>*>(om + i) = a;
            *reinterpret_cast<Vec<float, 4>*>(ov + i) = b;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j < n) {
                    om[i + j] = a.e[j];
                    ov[i + j] = b.e[j];
                }
        }
    }
}

static bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

template <typename P, typename G>
static void launch(cudaStream_t s, int bits, const Table& t, const Hyper& h, const Consts& c,
                   int chunk, unsigned blocks) {
    if (bits == 8) step8_kernel<P, G><<<blocks, THREADS, 0, s>>>(t, h, c, chunk);
    else step32_kernel<P, G><<<blocks, THREADS, 0, s>>>(t, h, c, chunk);
    FDB_LAUNCH_CHECK();
}
template <typename P>
static void launch_g(cudaStream_t s, int gtype, int bits, const Table& t, const Hyper& h,
                     const Consts& c, int chunk, unsigned blocks) {
    if (gtype == FDB_DTYPE_F32) launch<P, float>(s, bits, t, h, c, chunk, blocks);
    else if (gtype == FDB_DTYPE_BF16) launch<P, __nv_bfloat16>(s, bits, t, h, c, chunk, blocks);
    else launch<P, __half>(s, bits, t, h, c, chunk, blocks);
}

void step(cudaStream_t s, int sms, const fdb_adamw_tensor* ts, size_t count,
          const fdb_adamw_opts& o) {
    Hyper h{};
    h.lr = o.lr, h.b1 = o.beta1, h.b2 = o.beta2, h.wd = o.weight_decay;
    h.eps = (float)o.eps, h.grad_scale = (float)o.grad_scale;
    h.step = o.step, h.seed = o.seed;
    h.d_lr = o.d_lr, h.d_grad_scale = o.d_grad_scale, h.d_step = o.d_step;
    h.on_device = o.d_lr || o.d_step || o.d_grad_scale;
    const Consts c = consts_of(h, h.lr, std::max<int64_t>(h.step, 1), h.grad_scale);
    size_t total = 0;
    for (size_t i = 0; i < count; ++i) total += ts[i].n;
    const int chunk = total < (size_t)CHUNK * 4 * sms ? SMALL_CHUNK : CHUNK;
    // vectors of 4 (f32 moments) or 8 (8-bit) elements, 16 bytes at most
    const size_t per = o.state_bits == 8 ? 8 : 4;
    auto vec = [&](int dtype) {
        return std::min<size_t>(16, per * (dtype == FDB_DTYPE_F32 ? 4 : 2));
    };
    Table t;
    t.count = 0;
    unsigned blocks = 0;
    auto flush = [&] {
        if (t.count == 0) return;
        if (o.param_dtype == FDB_DTYPE_F32) launch_g<float>(s, o.grad_dtype, o.state_bits, t, h, c, chunk, blocks);
        else if (o.param_dtype == FDB_DTYPE_BF16)
            launch_g<__nv_bfloat16>(s, o.grad_dtype, o.state_bits, t, h, c, chunk, blocks);
        else launch_g<__half>(s, o.grad_dtype, o.state_bits, t, h, c, chunk, blocks);
        t.count = 0;
        blocks = 0;
    };
    for (size_t i = 0; i < count; ++i) {
        const fdb_adamw_tensor& x = ts[i];
        if (x.n == 0) continue;
        const size_t need = (x.n + chunk - 1) / chunk;
        if (t.count == TENSORS || need + blocks > 0x7fffffffu) flush();
        Entry& e = t.e[t.count++];
        e.p = x.param, e.g = x.grad, e.m = x.m, e.v = x.v, e.ms = x.m_scale, e.vs = x.v_scale;
        e.n = x.n;
        e.first = blocks;
        e.ordinal = (unsigned)i;
        const size_t sv = o.state_bits == 8 ? 8 : 16;
        e.wide = aligned(x.param, vec(o.param_dtype)) && aligned(x.grad, vec(o.grad_dtype)) &&
                 aligned(x.m, sv) && aligned(x.v, sv);
        blocks += (unsigned)need;
    }
    flush();
}

void values(cudaStream_t s, int sms, const int8_t* m, const float* ms, const uint8_t* v,
            const float* vs, size_t n, float* om, float* ov) {
    if (n == 0) return;
    const size_t blocks = (n + THREADS * 4 - 1) / (THREADS * 4);
    const int wide = aligned(m, 4) && aligned(v, 4) && aligned(om, 16) && aligned(ov, 16);
    values_kernel<<<(unsigned)std::min<size_t>(blocks, (size_t)sms * 16), THREADS, 0, s>>>(
        m, ms, v, vs, n, om, ov, wide);
    FDB_LAUNCH_CHECK();
}

}  // namespace adamw
}  // namespace fdb
