// Element types of the float operators: conversions between storage types and 32-bit floats, and 8-value
// loads and stores (vector where the caller found the rows aligned, by element otherwise).
#pragma once
#include "vela_b200.h"
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace vela {

template <class T> struct Elem;
template <> struct Elem<__nv_bfloat16> {
    static constexpr int code = VELA_T_BF16;
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Elem<__half> {
    static constexpr int code = VELA_T_F16;
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <> struct Elem<float> {
    static constexpr int code = VELA_T_F32;
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};

// v[i] = p[i] for i < n <= 8, 0 beyond; `vec`: n == 8 and p aligned to its 8 elements (at most 16 bytes)
template <class T> __device__ __forceinline__ void load8(const T* p, int n, bool vec, float (&v)[8]) {
    if (vec) {
        constexpr int W = sizeof(T) * 8 / 16;        // 16-byte words
        union { uint4 u[W]; T e[8]; } x;
#pragma unroll
        for (int i = 0; i < W; ++i) x.u[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = Elem<T>::get(x.e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? Elem<T>::get(p[i]) : 0.f;
    }
}
template <class T> __device__ __forceinline__ void store8(T* p, int n, bool vec, const float (&v)[8]) {
    if (vec) {
        constexpr int W = sizeof(T) * 8 / 16;
        union { uint4 u[W]; T e[8]; } x;
#pragma unroll
        for (int i = 0; i < 8; ++i) x.e[i] = Elem<T>::put(v[i]);
#pragma unroll
        for (int i = 0; i < W; ++i) reinterpret_cast<uint4*>(p)[i] = x.u[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) if (i < n) p[i] = Elem<T>::put(v[i]);
    }
}

// the larger of two, a NaN where either is one
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
inline size_t elem_bytes(int type) { return type == VELA_T_F32 ? 4 : type == VELA_T_I8 || type == VELA_T_E4M3 ? 1 : 2; }
}  // namespace vela
