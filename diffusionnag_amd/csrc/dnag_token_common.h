// What the token operators' kernels share (dnag_embed, dnag_block_norms, dnag_distill, dnag_sample .hip): element types, eight-element pieces of a row, sums and maxima
// over the lanes that hold one row, the launch helpers and the error path.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stddef.h>
#include "../../include/dnag.h"
#include "dnag_lds_limit.h"

// defined in dnag_lib.hip: formats dnag_last_error() of the calling thread and returns `code`
__attribute__((visibility("hidden"))) int dnag_fail(int code, const char *fmt, ...);

#define TOK_TRY(expr)                                                                                              \
    do {                                                                                                           \
        hipError_t e_ = (expr);                                                                                    \
        if (e_ != hipSuccess) return dnag_fail(DNAG_E_HIP, "%s failed: %s", #expr, hipGetErrorString(e_));        \
    } while (0)

typedef __bf16 tbf16;
typedef _Float16 tf16;
typedef float f8 __attribute__((ext_vector_type(8)));
template <class T> struct Vec8 { typedef T type __attribute__((ext_vector_type(8))); };

// Eight consecutive elements of a row as fp32.  The pointer needs the element's own alignment only (rows of odd width start
// anywhere): global memory takes 16-byte accesses at any address on this chip, and the copy compiles to them.
template <class T> __device__ __forceinline__ typename Vec8<T>::type load8_raw(const T *p) {
    typename Vec8<T>::type v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
}
template <class T> __device__ __forceinline__ f8 widen(typename Vec8<T>::type v) { return __builtin_convertvector(v, f8); }
template <class T> __device__ __forceinline__ f8 load8(const T *p) { return widen<T>(load8_raw(p)); }
// the first n of them as they are, zeros behind.  Not widened here: a conversion inside the branch would wait for the load there,
// and several of these in a row would wait one after the other (block norms' gradient, four rows to read: 146 us instead of 139).
template <class T> __device__ __forceinline__ typename Vec8<T>::type load8_raw_n(const T *p, int n) {
    typename Vec8<T>::type v;
    if (n >= 8) v = load8_raw(p);
    else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < n ? p[e] : (T)0.f;
    }
    return v;
}
// the first n (1..8) of them, `fill` behind
template <class T> __device__ __forceinline__ f8 load8_n(const T *p, int n, float fill = 0.f) {
    if (n >= 8) return load8(p);
    f8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? (float)p[e] : fill;
    return v;
}
template <class T> __device__ __forceinline__ void store8(T *p, f8 v) {
    const typename Vec8<T>::type o = __builtin_convertvector(v, typename Vec8<T>::type);      // one rounding, to nearest even
    __builtin_memcpy(p, &o, sizeof(o));
}
template <class T> __device__ __forceinline__ void store8_n(T *p, f8 v, int n) {
    if (n >= 8) { store8(p, v); return; }
#pragma unroll
    for (int e = 0; e < 8; ++e) if (e < n) p[e] = (T)v[e];
}
__device__ __forceinline__ f8 splat8(float x) { return f8{x, x, x, x, x, x, x, x}; }
__device__ __forceinline__ float sum8(f8 v) { return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7])); }
__device__ __forceinline__ float max8(f8 v) {
    return fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
}
// element `i` of an array that is fp32 or of type T, by a flag that is the same for the whole launch
template <class T> __device__ __forceinline__ f8 load8_either(const void *p, bool f32, size_t at, int n) {
    return f32 ? load8_n((const float *)p + at, n) : load8_n((const T *)p + at, n);
}
template <class T> __device__ __forceinline__ void store8_either(void *p, bool f32, size_t at, f8 v, int n) {
    if (f32) store8_n((float *)p + at, v, n);
    else store8_n((T *)p + at, v, n);
}

// p[a step] + p[(a + 1) step] + ... + p[(b - 1) step], in this order; sixteen loads are under way at a time, the last ones too (the
// remainder of an unrolled loop would wait for each)
__device__ __forceinline__ float sum_strided(const float *p, int a, int b, size_t step) {
    float s = 0.f;
    for (int k = a; k < b; k += 16) {
        float x[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) x[u] = p[(size_t)(k + u < b ? k + u : b - 1) * step];
#pragma unroll
        for (int u = 0; u < 16; ++u) s += k + u < b ? x[u] : 0.f;
    }
    return s;
}
// sum over the TPR lanes (a power of two <= 64, aligned) of a team; every lane gets the result, in one fixed order
template <int TPR> __device__ __forceinline__ float team_sum(float v) {
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
template <int TPR> __device__ __forceinline__ float team_max(float v) {
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

static inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
static inline int pow2_at_least(int64_t v, int lo, int hi) { int p = lo; while (p < hi && p < v) p *= 2; return p; }
static inline bool dtype_known(int t) { return t == DNAG_F32 || t == DNAG_BF16 || t == DNAG_F16; }
static inline size_t dtype_bytes(int t) { return t == DNAG_F32 ? 4 : 2; }
static inline size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// a grid holds less than 2^32 lanes along x
static inline int grid_fits(int64_t blocks, int64_t threads) {
    return blocks * threads < (1ll << 32) ? 0 : dnag_fail(DNAG_E_ARG, "%lld workgroups of %lld lanes: too many rows for one launch", (long long)blocks, (long long)threads);
}

// orders LDS accesses of a wave's lanes against each other (they run in step; this keeps the compiler from moving them)
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
