// Element types of the float operators: conversions between storage types and 32-bit floats, and 8-value loads and stores (vector
// where the caller found the rows aligned, by element otherwise).
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

// 8 neighbouring values as they lie in memory
template <class T> union Raw8 {
    uint4 u[sizeof(T) / 2];
    T e[8];
    __device__ __forceinline__ Raw8() {}
};
// p[i] for i < n <= 8, zero bits beyond; `vec`: n == 8 and p aligned to 16 bytes
template <class T> __device__ __forceinline__ void load_raw(Raw8<T>& x, const T* p, int n, bool vec) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < int(sizeof(T) / 2); ++i) x.u[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < int(sizeof(T) / 2); ++i) x.u[i] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int i = 0; i < 8; ++i) if (i < n) x.e[i] = p[i];
    }
}
// A warp's 256 neighbouring elements (as bits E) in rows that have their type's alignment only: lane l loads and stores elements l,
// l + 32, ..., so that a warp's 32 lie side by side; `line` (256 elements, the warp's own) brings them into the lanes' order, 8
// neighbours each, and back. p: the warp's first element; n: the elements that exist from there on (any number).
template <class E> union Line8 { uint4 u[(sizeof(E) + 1) / 2]; uint2 h; uint32_t w[2 * sizeof(E)]; E e[8]; };
template <class E> __device__ __forceinline__ void line_load(Line8<E>& x, const E* p, int n, int lane) {
#pragma unroll
    for (int k = 0; k < 8; ++k) x.e[k] = 32 * k + lane < n ? p[32 * k + lane] : E(0);
}
template <class E> __device__ __forceinline__ void line_to_lanes(Line8<E>& x, E* line, int lane) {
    static_assert(sizeof(E) >= 2, "16-byte loads");
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 8; ++k) line[32 * k + lane] = x.e[k];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < int(sizeof(E) / 2); ++i) x.u[i] = reinterpret_cast<const uint4*>(line + 8 * lane)[i];
}
template <class E> __device__ __forceinline__ void line_store(const Line8<E>& x, E* p, int n, E* line, int lane) {
    __syncwarp();
    if constexpr (sizeof(E) == 1) *reinterpret_cast<uint2*>(line + 8 * lane) = x.h;
    else
#pragma unroll
        for (int i = 0; i < int(sizeof(E) / 2); ++i) reinterpret_cast<uint4*>(line + 8 * lane)[i] = x.u[i];
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 8; ++k) if (32 * k + lane < n) p[32 * k + lane] = line[32 * k + lane];
}
// x as floats
template <class T> __device__ __forceinline__ void unpack8(float (&v)[8], const Raw8<T>& x) {
    if constexpr (Elem<T>::code == VELA_T_BF16) {
        const uint32_t w[4] = {x.u[0].x, x.u[0].y, x.u[0].z, x.u[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    } else if constexpr (Elem<T>::code == VELA_T_F16) {
        const uint32_t w[4] = {x.u[0].x, x.u[0].y, x.u[0].z, x.u[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i])); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = Elem<T>::get(x.e[i]);
    }
}

// the same as floats
template <class T> __device__ __forceinline__ void load8(const T* p, int n, bool vec, float (&v)[8]) {
    Raw8<T> x;
    load_raw(x, p, n, vec);
    unpack8(v, x);
}
// v as T, two at a time where T is narrower than a float (one instruction then)
template <class T> __device__ __forceinline__ void pack8(Raw8<T>& x, const float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (Elem<T>::code == VELA_T_BF16) { const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t*>(&p); }
            else { const __half2 p = __floats2half2_rn(v[2 * i], v[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t*>(&p); }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x.e[i] = Elem<T>::put(v[i]);
    }
}
template <class T> struct Bits { typedef uint16_t E; };
template <> struct Bits<float> { typedef uint32_t E; };
template <class T> __device__ __forceinline__ void store8(T* p, int n, bool vec, const float (&v)[8]) {
    Raw8<T> x;
    pack8(x, v);
    if (vec) {
#pragma unroll
        for (int i = 0; i < int(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = x.u[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) if (i < n) p[i] = x.e[i];
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
