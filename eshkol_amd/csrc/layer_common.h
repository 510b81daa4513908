/*
 * What the layer kernels (layernorm.hip, linear_16.hip) share: element types,
 * 16-byte vectors of them at any alignment, reductions, and the checks of a call.
 */
#ifndef ESHKOL_HIP_LAYER_COMMON_H
#define ESHKOL_HIP_LAYER_COMMON_H

#include "hip_common.h"
#include "eshkol/backend/gpu/gpu_hip_layers.h"

#include <math.h>

/* Says why a call is refused (ESHKOL_GPU_VERBOSE=1) and refuses it. */
#define LAYER_REFUSE(name, fmt, ...) do { GPU_LOG("%s: " fmt, name, ##__VA_ARGS__); return -1; } while (0)

/* Makes the stream's device current for the length of a call. The null stream
 * belongs to the current device. */
struct EshkolStreamDevice {
    int before = -1;
    bool ok = true;
    explicit EshkolStreamDevice(hipStream_t st) {
        if (!st) return;
        int dev = 0, now = 0;
        if (hipStreamGetDevice(st, &dev) != hipSuccess || hipGetDevice(&now) != hipSuccess) { ok = false; return; }
        if (dev != now) { before = now; ok = hipSetDevice(dev) == hipSuccess; }
    }
    ~EshkolStreamDevice() { if (before >= 0) (void)hipSetDevice(before); }
    EshkolStreamDevice(const EshkolStreamDevice&) = delete;
    EshkolStreamDevice& operator=(const EshkolStreamDevice&) = delete;
};

static inline size_t layer_dtype_size(int dtype) { return dtype == 0 ? 8 : dtype == 1 ? 4 : 2; }
/* a pointer on an element's boundary */
static inline bool layer_aligned(const void* p, int dtype) { return ((uintptr_t)p & (layer_dtype_size(dtype) - 1)) == 0; }
static inline bool layer_param_ok(int dtype, int param) { return param == dtype || (param == 1 && (dtype == 2 || dtype == 3)); }

#ifdef __HIPCC__

namespace layer {

template <int DT> struct Elem;
template <> struct Elem<0> { typedef double T; typedef double Acc; };
template <> struct Elem<1> { typedef float T; typedef float Acc; };
template <> struct Elem<2> { typedef _Float16 T; typedef float Acc; };
template <> struct Elem<3> { typedef __bf16 T; typedef float Acc; };

/* 16 bytes of elements; the alignment it promises is an element's, which is all the
 * rows have (global memory takes 16-byte accesses at any address) */
template <class T> struct Vec16 {
    static constexpr int N = 16 / (int)sizeof(T);
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

/* elements c .. c + N - 1 of a row of n, zeros beyond its end; EVEN: the caller knows that they are all there */
template <class T, class Acc, int N, bool EVEN = false>
__device__ __forceinline__ void load_row(const T* row, uint32_t c, uint32_t n, Acc (&out)[N]) {
    if (EVEN || c + N <= n) {
        typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
        const vec v = *(const vec*)(row + c);
#pragma unroll
        for (int e = 0; e < N; e++) out[e] = (Acc)v[e];
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) out[e] = c + e < n ? (Acc)row[c + e] : (Acc)0;
    }
}

template <class T, class Acc, int N, bool STREAM = false>
__device__ __forceinline__ void store_row(T* row, uint32_t c, uint32_t n, const Acc (&in)[N]) {
    if (c + N <= n) {
        typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
        vec v;
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = (T)in[e];
        if constexpr (STREAM) __builtin_nontemporal_store(v, (vec*)(row + c));
        else *(vec*)(row + c) = v;
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) if (c + e < n) row[c + e] = (T)in[e];
    }
}

/* a parameter vector of type T, or of fp32 where wide != 0; `none` for a NULL one */
template <class T, class Acc, int N, bool EVEN = false>
__device__ __forceinline__ void load_param(const void* p, int wide, Acc none, uint32_t c, uint32_t n, Acc (&out)[N]) {
    if (!p) {
#pragma unroll
        for (int e = 0; e < N; e++) out[e] = none;
    } else if (wide) load_row<float, Acc, N, EVEN>((const float*)p, c, n, out);
    else load_row<T, Acc, N, EVEN>((const T*)p, c, n, out);
}

template <class Acc> __device__ __forceinline__ Acc fma_of(Acc a, Acc b, Acc c);
template <> __device__ __forceinline__ float fma_of(float a, float b, float c) { return fmaf(a, b, c); }
template <> __device__ __forceinline__ double fma_of(double a, double b, double c) { return fma(a, b, c); }

/* the wave's sum, in every lane */
template <class Acc> __device__ __forceinline__ Acc wave_sum(Acc v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

}  // namespace layer
#endif
#endif
