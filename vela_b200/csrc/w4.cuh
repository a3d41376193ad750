// 4-bit weight tiles on the tensor cores: the 16 x 64 tile of vela_w4 (512 bytes, 16 per lane) against up to
// 8 NT activation rows.
//
// Lane 4 g + t of a warp holds, in word j (j < 4) of its 16 bytes, rows g and g + 8 at the four columns
// k = 32 (j / 2) + 8 t + 4 (j % 2) + {0, 1, 2, 3}.  A product over k does not mind in which order k runs, so those
// columns stand in the places that the instruction numbers 2t, 2t + 1, 2t + 8, 2t + 9 (16-bit operands) or 4t .. 4t + 3
// (8-bit ones), for the weights and the activations alike: each lane reads 8 neighbouring activations at a time, and
// the codes come out of a word by masks.  With words w0..w3 of nibbles 0..7, nibbles (0, 4) and (2, 6) are row g's,
// (1, 5) and (3, 7) row g + 8's column pairs (0, 1) and (2, 3).
//
// 16-bit operands: 0x4300 | n is the bf16 number 128 + n and 0x6400 | n the f16 number 1024 + n, from which 128 + zero
// (1024 + zero) is taken exactly, so the operand is the integer code - zero and no rounding happens before the 32-bit
// accumulation.  8-bit operands: the codes go in as unsigned bytes, and zero times the sum of the activations
// (one more product, by ones) is taken off the 32-bit integer sum.
#pragma once
#include "elem.cuh"
#include "vela_b200.h"

namespace vela {
namespace w4 {

constexpr int TILE_ROWS = 16, TILE_K = 64, TILE_BYTES = 512;

struct Weights {                     // one matrix on the device
    const uint4* q; const uint32_t* scale; const uint16_t* zero;     // scale, zero: pairs (row g, row g + 8)
    int N, K, kt, ng, gshift;        // kt: tiles along K; ng: groups; gshift: log2(group)
    bool f16;                        // scale type
};

__device__ __forceinline__ void mma_f32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_i8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <class T> struct Magic;
template <> struct Magic<__nv_bfloat16> {
    static constexpr uint32_t bits = 0x43004300u, one = 0x00010001u, base = 0x43004300u;
    static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
        __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
        return *reinterpret_cast<uint32_t*>(&r);
    }
};
template <> struct Magic<__half> {
    static constexpr uint32_t bits = 0x64006400u, one = 0x00010001u, base = 0x64006400u;
    static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
        __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
        return *reinterpret_cast<uint32_t*>(&r);
    }
};

// the pair (row g, row g + 8) of scales as floats
__device__ __forceinline__ float2 scale_pair(uint32_t u, bool f16) {
    if (f16) return __half22float2(*reinterpret_cast<__half2*>(&u));
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// Activation types.  X: what lies in memory; M: the operand type of the product.  `half` loads the 8 activations of a
// lane in one half tile as the registers of its two products' second operands.
template <int XT> struct Act;
template <> struct Act<VELA_T_BF16> {
    typedef __nv_bfloat16 X; typedef __nv_bfloat16 M; static constexpr bool scaled = false, integer = false; static constexpr int regs = 4;
};
template <> struct Act<VELA_T_F16> {
    typedef __half X; typedef __half M; static constexpr bool scaled = false, integer = false; static constexpr int regs = 4;
};
template <> struct Act<VELA_T_E4M3> {
    typedef uint8_t X; typedef __half M; static constexpr bool scaled = true, integer = false; static constexpr int regs = 4;
};
template <> struct Act<VELA_T_I8> {
    typedef uint8_t X; typedef int8_t M; static constexpr bool scaled = true, integer = true; static constexpr int regs = 2;
};

// p[0 .. n) with zeros beyond, n <= 8 (may be negative); p null: zeros
template <int XT> __device__ __forceinline__ void load_half(uint32_t (&b)[Act<XT>::regs], const typename Act<XT>::X* p, int n, bool vec) {
    if constexpr (sizeof(typename Act<XT>::X) == 2) {
        if (!p || n <= 0) { b[0] = b[1] = b[2] = b[3] = 0u; return; }
        if (vec) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
            b[0] = u.x; b[1] = u.y; b[2] = u.z; b[3] = u.w;
        } else {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                b[i] = 2 * i < n ? h[2 * i] : 0u;
                if (2 * i + 1 < n) b[i] |= uint32_t(h[2 * i + 1]) << 16;
            }
        }
    } else {
        uint2 u = make_uint2(0u, 0u);
        if (p && n > 0) {
            if (vec) u = __ldg(reinterpret_cast<const uint2*>(p));
            else {
#pragma unroll
                for (int i = 0; i < 4; ++i) { if (i < n) u.x |= uint32_t(p[i]) << (8 * i); if (i + 4 < n) u.y |= uint32_t(p[i + 4]) << (8 * i); }
            }
        }
        if constexpr (XT == VELA_T_I8) {         // bytes in the order of a word's codes: columns 0, 2, 1, 3
            b[0] = __byte_perm(u.x, 0u, 0x3120);
            b[1] = __byte_perm(u.y, 0u, 0x3120);
        } else {
            const uint32_t w[2] = {u.x, u.y};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
                b[i] = uint32_t(h.x) | uint32_t(h.y) << 16;
            }
        }
    }
}

// One half tile (words u0, u1 = 32 columns) of 16 rows against 8 activation rows, added to c; zz: 128 + zero as bf16
// pairs (1024 + zero as f16 pairs) of rows g and g + 8.
template <class M> __device__ __forceinline__ void decode16(uint32_t (&a)[4], uint32_t u, uint32_t z0, uint32_t z1) {
    constexpr uint32_t m = 0x000f000fu, b = Magic<M>::bits;
    a[0] = Magic<M>::sub((u & m) | b, z0);
    a[1] = Magic<M>::sub(((u >> 4) & m) | b, z1);
    a[2] = Magic<M>::sub(((u >> 8) & m) | b, z0);
    a[3] = Magic<M>::sub(((u >> 12) & m) | b, z1);
}

// The running product of R row tiles with 8 NT activation rows.  c0, c1: row g, activation rows 2t and 2t + 1; c2, c3: row g + 8.
template <int XT, int NT, int R> struct Acc {
    float v[R][NT][4];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[r][n][i] = 0.f;
    }
};

struct ScaleZero { uint32_t s; uint32_t z; };
__device__ __forceinline__ ScaleZero load_scale(const Weights& W, int rt, int k, int g) {
    const size_t i = (size_t(rt) * W.ng + (k >> W.gshift)) * 8 + g;
    ScaleZero r;
    r.s = __ldg(W.scale + i);
    r.z = W.zero ? __ldg(W.zero + i) : 0x0808u;
    return r;
}

// Adds one 64-column tile of row tile r to acc.  b: the activations' operands [half][NT].  sx (8-bit activations): the
// scales of activation rows 2t, 2t + 1.  G32: groups of 32 columns, so each half has its own scales.
template <int XT, int NT, bool G32>
__device__ __forceinline__ void tile(float (&acc)[NT][4], const uint4& w, const uint32_t (&b)[2][NT][Act<XT>::regs], const int (&ones)[2][NT][2],
                                     const ScaleZero (&sz)[2], const float2 (&sx)[NT], bool f16) {
    typedef typename Act<XT>::M M;
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    if constexpr (Act<XT>::integer) {
        int c[NT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (G32 || h == 0) {
#pragma unroll
                for (int n = 0; n < NT; ++n) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0;
            }
            constexpr uint32_t m = 0x0f0f0f0fu;
            const uint32_t a0 = u[2 * h] & m, a1 = (u[2 * h] >> 4) & m, a2 = u[2 * h + 1] & m, a3 = (u[2 * h + 1] >> 4) & m;
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_i8(c[n], a0, a1, a2, a3, b[h][n][0], b[h][n][1]);
            if (G32 || h == 1) {
                const ScaleZero q = sz[G32 ? h : 0];
                const float2 s = scale_pair(q.s, f16);
                const int z0 = q.z & 0xff, z1 = q.z >> 8;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int t0 = ones[h][n][0] + (G32 ? 0 : ones[0][n][0]), t1 = ones[h][n][1] + (G32 ? 0 : ones[0][n][1]);
                    acc[n][0] = fmaf(s.x * sx[n].x, float(c[n][0] - z0 * t0), acc[n][0]);
                    acc[n][1] = fmaf(s.x * sx[n].y, float(c[n][1] - z0 * t1), acc[n][1]);
                    acc[n][2] = fmaf(s.y * sx[n].x, float(c[n][2] - z1 * t0), acc[n][2]);
                    acc[n][3] = fmaf(s.y * sx[n].y, float(c[n][3] - z1 * t1), acc[n][3]);
                }
            }
        }
    } else {
        float c[NT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (G32 || h == 0) {
#pragma unroll
                for (int n = 0; n < NT; ++n) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.f;
            }
            const ScaleZero q = sz[G32 ? h : 0];
            // 128 + zero (1024 + zero) lies zero steps above the base, in both halves of the pair
            const uint32_t z0 = Magic<M>::base + Magic<M>::one * (q.z & 0xff), z1 = Magic<M>::base + Magic<M>::one * (q.z >> 8);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t a[4];
                decode16<M>(a, u[2 * h + j], z0, z1);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_f32(c[n], a, b[h][n][2 * j], b[h][n][2 * j + 1], M());
            }
            if (G32 || h == 1) {
                const float2 s = scale_pair(q.s, f16);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if constexpr (Act<XT>::scaled) {
                        acc[n][0] = fmaf(s.x * sx[n].x, c[n][0], acc[n][0]);
                        acc[n][1] = fmaf(s.x * sx[n].y, c[n][1], acc[n][1]);
                        acc[n][2] = fmaf(s.y * sx[n].x, c[n][2], acc[n][2]);
                        acc[n][3] = fmaf(s.y * sx[n].y, c[n][3], acc[n][3]);
                    } else {
                        acc[n][0] = fmaf(s.x, c[n][0], acc[n][0]);
                        acc[n][1] = fmaf(s.x, c[n][1], acc[n][1]);
                        acc[n][2] = fmaf(s.y, c[n][2], acc[n][2]);
                        acc[n][3] = fmaf(s.y, c[n][3], acc[n][3]);
                    }
                }
            }
        }
    }
}

// sums of the integer activations of one half tile for activation rows 2t, 2t + 1
template <int XT, int NT> __device__ __forceinline__ void sums(int (&ones)[2][NT][2], const uint32_t (&b)[2][NT][Act<XT>::regs]) {
    if constexpr (Act<XT>::integer) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                int c[4] = {0, 0, 0, 0};
                mma_i8(c, 0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u, b[h][n][0], b[h][n][1]);
                ones[h][n][0] = c[0]; ones[h][n][1] = c[1];
            }
    }
}

}  // namespace w4

// checks a descriptor and brings it into the kernels' form; `name` begins the messages
w4::Weights w4_weights(const vela_w4& w, const char* name);
inline size_t w4_bytes(int N, int K) { return (size_t(N) + 15) / 16 * ((size_t(K) + 63) / 64) * 512; }
inline size_t w4_scales(int N, int K, int group) { return (size_t(N) + 15) / 16 * 16 * ((size_t(K) + group - 1) / group); }
inline bool w4_sizes_ok(int N, int K, int group) { return N > 0 && K > 0 && N <= (1 << 30) && K <= (1 << 30) && (group == 32 || group == 64 || group == 128); }
}  // namespace vela
