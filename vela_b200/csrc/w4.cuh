// 4-bit weight tiles on the tensor cores: the 16 x 64 tile of vela_w4 (512 bytes, 16 per lane) against up to 8 NT activation rows.
//
// Lane 4 g + t of a warp holds, in word j (j < 4) of its 16 bytes, rows g and g + 8 at the four columns k = 32 (j / 2) + 8 t + 4 (j
// % 2) + {0, 1, 2, 3}.  A product over k does not mind in which order k runs, so those columns stand in the places that the
// instruction numbers 2t, 2t + 1, 2t + 8, 2t + 9 (16-bit operands) or 4t .. 4t + 3 (8-bit ones), for the weights and the
// activations alike.  Of a word's nibbles 0..7, (0, 4) and (2, 6) are row g's column pairs (0, 1) and (2, 3), (1, 5) and (3, 7) row
// g + 8's.
//
// 16-bit operands: 0x4300 | n is the bf16 number 128 + n and 0x6400 | n the f16 number 1024 + n (0x5400 | n << 4 the number 64 + n,
// which saves a shift), from which 128 + zero (1024 + zero, 64 + zero) is taken exactly: the operand is the integer code - zero,
// and nothing is rounded before the 32-bit accumulation.  8-bit operands: a mask leaves the unsigned byte code (row g) or 16 * code
// (row g + 8), and zero times the sum of the activations, from one more product by ones, is taken off the 32-bit integer sum.
#pragma once
#include "elem.cuh"
#include "vela_b200.h"

namespace vela {
namespace w4 {

struct Weights {                     // one matrix (or several, one after another) on the device
    const uint4* q; const uint32_t* scale; const uint16_t* zero;     // scale, zero: pairs (row g, row g + 8)
    int N, K, kt, ng, gshift;        // kt: tiles along K; ng: groups; gshift: log2(group)
    bool f16;                        // scale type
};
__host__ __device__ __forceinline__ int row_tiles(const Weights& W) { return (W.N + 15) >> 4; }
__host__ __device__ __forceinline__ int units(const Weights& W) { return (W.kt + 1) >> 1; }

template <class M> struct Ops;      // M: the operands' type
template <> struct Ops<__nv_bfloat16> {
    static constexpr uint32_t base0 = 0x43004300u, base1 = 0x43004300u;      // of rows g and g + 8
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
        __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
        return *reinterpret_cast<uint32_t*>(&r);
    }
    static __device__ __forceinline__ uint32_t high(uint32_t u, uint32_t, uint32_t m, uint32_t k) { return and_or(u >> 4, m, k); }
    static __device__ __forceinline__ uint32_t and_or(uint32_t u, uint32_t m, uint32_t k) {
        uint32_t d;
        asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(u), "r"(m), "r"(k));
        return d;
    }
    static constexpr uint32_t zstep1 = 1;                  // what a step of the zero point adds to the number's bits
};
template <> struct Ops<__half> {
    static constexpr uint32_t base0 = 0x64006400u, base1 = 0x54005400u;
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
        __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
        return *reinterpret_cast<uint32_t*>(&r);
    }
    static __device__ __forceinline__ uint32_t high(uint32_t u, uint32_t m4, uint32_t, uint32_t k) { return Ops<__nv_bfloat16>::and_or(u, m4, k); }
    static __device__ __forceinline__ uint32_t and_or(uint32_t u, uint32_t m, uint32_t k) { return Ops<__nv_bfloat16>::and_or(u, m, k); }
    static constexpr uint32_t zstep1 = 16;
};
__device__ __forceinline__ void mma_i8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Masks and bases in registers that the compiler does not see through: an instruction takes one constant at most, so as constants
// the mask and the base would cost a second instruction for each operand.
struct Consts { uint32_t m, m4, k0, k1; };
template <class M> __device__ __forceinline__ Consts consts() {
    Consts c;
    asm volatile("mov.b32 %0, 0x000f000f;" : "=r"(c.m));
    asm volatile("mov.b32 %0, 0x00f000f0;" : "=r"(c.m4));
    asm volatile("mov.b32 %0, %1;" : "=r"(c.k0) : "n"(Ops<M>::base0));
    asm volatile("mov.b32 %0, %1;" : "=r"(c.k1) : "n"(Ops<M>::base1));
    return c;
}
template <> __device__ __forceinline__ Consts consts<int8_t>() { return Consts{}; }

// a / b for a >= 0, b > 0: the quotient of floats is off by a few at most, which the loops put right (a division of integers takes
// many times as long)
__device__ __forceinline__ int quot(int a, int b) {
    int q = int(__fdividef(float(a), float(b))), r = a - q * b;
    while (r < 0) { --q; r += b; }
    while (r >= b) { ++q; r -= b; }
    return q;
}

// the pair (row g, row g + 8) of scales as floats
__device__ __forceinline__ float2 scale_pair(uint32_t u, bool f16) {
    if (f16) return __half22float2(*reinterpret_cast<__half2*>(&u));
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// weights pass through once: they leave the L1 cache to others
__device__ __forceinline__ uint4 load_tile(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// A unit is two neighbouring tiles (128 columns) of one row tile: what a warp loads at once.  FOLD (32, 64 or 128) is the number of
// columns between scalings, the smaller of the weights' and the activations' group; a unit has one scale (and zero) for each fold.
template <int FOLD, bool ZERO> struct Unit {
    uint4 w[2];
    uint32_t s[128 / FOLD];
    uint32_t z[ZERO ? 128 / FOLD : 1];
};

// Where a unit of one row tile lies for one lane.
struct RowPtr { const uint4* q; const uint32_t* s; const uint16_t* z; };
__device__ __forceinline__ RowPtr row_ptr(const Weights& W, size_t rt, int u, int lane) {
    const size_t grp = rt * W.ng + (size_t(u) << (7 - W.gshift));
    RowPtr p;
    p.q = W.q + (rt * W.kt + 2 * size_t(u)) * 32 + lane;
    p.s = W.scale + grp * 8 + (lane >> 2);
    p.z = W.zero + grp * 8 + (lane >> 2);
    return p;
}
// `n` units on
__device__ __forceinline__ void advance(RowPtr& p, const Weights& W, int n) {
    p.q += n * 64;
    p.s += (n << (7 - W.gshift)) * 8;
    p.z += (n << (7 - W.gshift)) * 8;
}
template <int FOLD, bool ZERO> __device__ __forceinline__ void load_unit(Unit<FOLD, ZERO>& o, const RowPtr& p, const Weights& W) {
    o.w[0] = load_tile(p.q);
    o.w[1] = load_tile(p.q + 32);
#pragma unroll
    for (int f = 0; f < 128 / FOLD; ++f) {
        const int grp = FOLD == 64 ? (f * FOLD) >> W.gshift : f;      // FOLD 32 and 128 are the weights' own groups
        o.s[f] = __ldg(p.s + grp * 8);
        if constexpr (ZERO) o.z[f] = __ldg(p.z + grp * 8);
    }
}
// The last unit (number u) may lack its second tile or its last groups: the last tile and group are read again in their place, and
// meet activations of zero.
template <int FOLD, bool ZERO> __device__ __forceinline__ void load_last(Unit<FOLD, ZERO>& o, const RowPtr& p, const Weights& W, int u) {
    o.w[0] = load_tile(p.q);
    o.w[1] = load_tile(p.q + (2 * u + 1 < W.kt ? 32 : 0));
    const int left = W.ng - 1 - (u << (7 - W.gshift));
#pragma unroll
    for (int f = 0; f < 128 / FOLD; ++f) {
        const int grp = min((f * FOLD) >> W.gshift, left);
        o.s[f] = __ldg(p.s + grp * 8);
        if constexpr (ZERO) o.z[f] = __ldg(p.z + grp * 8);
    }
}

// Activation types.  X: what lies in memory; M: the operands' type; REGS: a lane's registers for the 8 columns that it takes of 32.
template <int XT> struct Act;
template <> struct Act<VELA_T_BF16> { typedef __nv_bfloat16 X; typedef __nv_bfloat16 M; static constexpr bool scaled = false, integer = false; static constexpr int REGS = 4; };
template <> struct Act<VELA_T_F16> { typedef __half X; typedef __half M; static constexpr bool scaled = false, integer = false; static constexpr int REGS = 4; };
template <> struct Act<VELA_T_E4M3> { typedef uint8_t X; typedef __half M; static constexpr bool scaled = true, integer = false; static constexpr int REGS = 4; };
template <> struct Act<VELA_T_I8> { typedef uint8_t X; typedef int8_t M; static constexpr bool scaled = true, integer = true; static constexpr int REGS = 2; };

// A lane's 8 activations p[0 .. 8) of a 32-column part as operands.  Not WHOLE: n of them exist (may be negative), zeros stand for
// the others, and p has its type's alignment only.  CONSTANT: nobody writes them while the kernel is there.
template <int XT, bool WHOLE, bool CONSTANT = true> __device__ __forceinline__ void load_x8(uint32_t (&b)[Act<XT>::REGS], const typename Act<XT>::X* p, int n) {
    static_assert(CONSTANT || sizeof(typename Act<XT>::X) == 2, "8-bit rows are always read as constants");
    if constexpr (sizeof(typename Act<XT>::X) == 2) {
        if constexpr (WHOLE) {
            const uint4 u = CONSTANT ? __ldg(reinterpret_cast<const uint4*>(p)) : *reinterpret_cast<const uint4*>(p);
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
        if constexpr (WHOLE) u = __ldg(reinterpret_cast<const uint2*>(p));
        else {
#pragma unroll
            for (int i = 0; i < 4; ++i) { if (i < n) u.x |= uint32_t(p[i]) << (8 * i); if (i + 4 < n) u.y |= uint32_t(p[i + 4]) << (8 * i); }
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

// Adds one unit of R row tiles to acc: c0, c1 = row g and activation rows 2t, 2t + 1; c2, c3 = row g + 8.  x[n]: this lane's place
// (row g of column tile n, column 8 t of the unit; any row where there is none: its column of the product is not used); WHOLE: all
// 128 columns exist and x is aligned to 8 of them, else left columns exist from x on; sx(f, n): the scales of activation rows 2t,
// 2t + 1 of column tile n in fold f (8-bit forms).
template <int XT, bool WHOLE, int NT, int R, bool CONSTANT = true, int FOLD, bool ZERO, class SX>
__device__ __forceinline__ void unit(float (&acc)[R][NT][4], const Unit<FOLD, ZERO> (&W)[R], const typename Act<XT>::X* const (&x)[NT], int left, bool f16,
                                     const Consts& k, SX sx) {
    typedef typename Act<XT>::M M;
    constexpr int HALVES = FOLD / 32;
    constexpr bool AHEAD = NT == 1;                        // all of the unit's activations at once, where the registers allow
    uint32_t all[AHEAD ? 4 : 1][NT][Act<XT>::REGS];
    if constexpr (AHEAD) {
#pragma unroll
        for (int h = 0; h < 4; ++h) load_x8<XT, WHOLE, CONSTANT>(all[h][0], x[0] + 32 * h, left - 32 * h);
    }
#pragma unroll
    for (int f = 0; f < 128 / FOLD; ++f) {
        float d[R][NT][4];
        float2 tot[NT];                                    // integer forms: sums of activation rows 2t, 2t + 1
        if constexpr (Act<XT>::integer) {
            int c[R][NT][4] = {}, s[NT][4] = {};
#pragma unroll
            for (int h = f * HALVES; h < (f + 1) * HALVES; ++h) {
                uint32_t b[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if constexpr (AHEAD) { b[n][0] = all[h][n][0]; b[n][1] = all[h][n][1]; }
                    else load_x8<XT, WHOLE, CONSTANT>(b[n], x[n] + 32 * h, left - 32 * h);
                    mma_i8(s[n], 0x01010101u, 0u, 0x01010101u, 0u, b[n][0], b[n][1]);
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const uint4 v = W[r].w[h >> 1];
                    const uint32_t u0 = h & 1 ? v.z : v.x, u1 = h & 1 ? v.w : v.y;
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_i8(c[r][n], u0 & 0x0f0f0f0fu, u0 & 0xf0f0f0f0u, u1 & 0x0f0f0f0fu, u1 & 0xf0f0f0f0u, b[n][0], b[n][1]);
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                tot[n] = make_float2(float(s[n][0]), float(s[n][1]));
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float z0 = ZERO ? float(W[r].z[ZERO ? f : 0] & 0xffu) : 8.f, z1 = ZERO ? float(W[r].z[ZERO ? f : 0] >> 8) : 8.f;
                    // exact: all of these are integers (or sixteenths) below 2^24
                    d[r][n][0] = fmaf(-z0, tot[n].x, float(c[r][n][0])); d[r][n][1] = fmaf(-z0, tot[n].y, float(c[r][n][1]));
                    d[r][n][2] = fmaf(0.0625f, float(c[r][n][2]), -z1 * tot[n].x); d[r][n][3] = fmaf(0.0625f, float(c[r][n][3]), -z1 * tot[n].y);
                }
            }
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int n = 0; n < NT; ++n) d[r][n][0] = d[r][n][1] = d[r][n][2] = d[r][n][3] = 0.f;
            uint32_t z0[R], z1[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {      // the number above, with the zero point added to its bits, in both halves
                const uint32_t z = ZERO ? W[r].z[ZERO ? f : 0] : 0x0808u;
                z0[r] = Ops<M>::base0 + 0x00010001u * (z & 0xffu);
                z1[r] = Ops<M>::base1 + 0x00010001u * Ops<M>::zstep1 * (z >> 8);
            }
#pragma unroll
            for (int h = f * HALVES; h < (f + 1) * HALVES; ++h) {
                uint32_t b[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if constexpr (AHEAD) { b[n][0] = all[h][n][0]; b[n][1] = all[h][n][1]; b[n][2] = all[h][n][2]; b[n][3] = all[h][n][3]; }
                    else load_x8<XT, WHOLE, CONSTANT>(b[n], x[n] + 32 * h, left - 32 * h);
                }
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const uint4 v = W[r].w[h >> 1];
                        const uint32_t u = h & 1 ? (j ? v.w : v.z) : (j ? v.y : v.x), u8 = u >> 8;
                        const uint32_t a[4] = {Ops<M>::sub(Ops<M>::and_or(u, k.m, k.k0), z0[r]), Ops<M>::sub(Ops<M>::high(u, k.m4, k.m, k.k1), z1[r]),
                                               Ops<M>::sub(Ops<M>::and_or(u8, k.m, k.k0), z0[r]), Ops<M>::sub(Ops<M>::high(u8, k.m4, k.m, k.k1), z1[r])};
#pragma unroll
                        for (int n = 0; n < NT; ++n) Ops<M>::mma(d[r][n], a, b[n][2 * j], b[n][2 * j + 1]);
                    }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float2 s = scale_pair(W[r].s[f], f16);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float2 p = make_float2(s.x, s.x), q = make_float2(s.y, s.y);
                if constexpr (Act<XT>::scaled) {
                    const float2 e = sx(f, n);
                    p = make_float2(s.x * e.x, s.x * e.y); q = make_float2(s.y * e.x, s.y * e.y);
                }
                acc[r][n][0] = fmaf(p.x, d[r][n][0], acc[r][n][0]);
                acc[r][n][1] = fmaf(p.y, d[r][n][1], acc[r][n][1]);
                acc[r][n][2] = fmaf(q.x, d[r][n][2], acc[r][n][2]);
                acc[r][n][3] = fmaf(q.y, d[r][n][3], acc[r][n][3]);
            }
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
