// Streaming row tiles of 4-bit weights past stationary activations, for products in which a block has many row tiles and the same
// few activation rows.
//
// A warp keeps the activations of UW units (128 columns each) in registers and streams row tiles past them, so they are read once
// for many row tiles.  They are f16 (exactly: f16 as it is, bf16 and float with a power of two for each row and 128 columns; floats
// as the sum of two).  The bits of a nibble at the bottom of a 16-bit half are, as they stand, the (subnormal) f16 number code *
// 2^-24, four bits up code * 2^-20, both exact and taken by the tensor cores at full rate: a word of 8 codes takes one shift and
// four masks and no conversion (w4.cuh's direct forms: 9 to 11).  Zero times the activations' sum is taken off the sum of products.
// A unit costs 3 loads, 40 instructions of decoding, 8 products and 12 to 16 for its scales.  While a block's loop runs it takes 41
// bytes of weights a nanosecond (6.1 TB/s over all SMs) in the one-term form; the two-term form has 16 products a unit in one
// chain and takes about half of that.
#pragma once
#include "w4.cuh"
#include "w4_plan.h"

namespace vela {
namespace w4 {

// asks for `bytes` (a multiple of 16) from p to be brought to the L2 cache
__device__ __forceinline__ void prefetch_l2(const void* p, uint32_t bytes) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" :: "l"(p), "r"(bytes) : "memory");
}

// ---------------------------------------------------------------- activations as operands
// F: f16 values.  H: the sum of two f16 values (22 bits).  regs: a lane's registers for one unit and 8 rows.
enum Kind { F, H };
template <Kind KIND> __host__ __device__ constexpr int regs() { return KIND == F ? 16 : 32; }
// For each fold and the lane's two columns of the product (rows 2t and 2t + 1 of the activations): the factor that the operands
// have lost, and their sum.
template <int FOLD> struct Pairs { float2 v[128 / FOLD][2]; };

// Fills in the pairs of H: the sums come out of a product by ones where they are needed, the factor (known to the four lanes of row
// g) by a shuffle.
template <int FOLD> __device__ __forceinline__ void make_pairs(Pairs<FOLD>& p, const uint32_t (&b)[32], int t, float lost) {
    constexpr int HALVES = FOLD / 32;
    const float e = __shfl_sync(0xffffffffu, lost, 8 * t), o = __shfl_sync(0xffffffffu, lost, 8 * t + 4);
#pragma unroll
    for (int f = 0; f < 128 / FOLD; ++f) {
        float c[4] = {};
        const uint32_t ones[4] = {0x3c003c00u, 0u, 0x3c003c00u, 0u};
#pragma unroll
        for (int h = f * HALVES; h < (f + 1) * HALVES; ++h)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                Ops<__half>::mma(c, ones, b[16 + 4 * h + 2 * j], b[16 + 4 * h + 2 * j + 1]);
                Ops<__half>::mma(c, ones, b[4 * h + 2 * j], b[4 * h + 2 * j + 1]);
            }
        p.v[f][0] = make_float2(e, c[0]); p.v[f][1] = make_float2(o, c[1]);
    }
}

// The power of two that brings a row's 128 values (top: the bits of the largest magnitude among a lane's 32) into f16's range, the
// largest to [2^14, 2^15), and its inverse.  bf16's 8 bits then fit exactly down to 2^-31 of the largest, and what is smaller is
// rounded to 2^-39 of it, below a 32-bit sum's own rounding.
__device__ __forceinline__ float2 row_scale(uint32_t top) {
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    int e = int(top >> 23) - 127;                          // 128: an infinity or a NaN, which stays one
    e = e > 127 ? 127 : e < -100 ? -100 : e;               // both factors are normal floats
    return make_float2(__uint_as_float(uint32_t(127 + 14 - e) << 23), __uint_as_float(uint32_t(127 - 14 + e) << 23));
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// One unit of a staged row (stage_unit): x this lane's row g from column 8 t of the unit on, e and o the unit's pairs of the rows
// 2t and 2t + 1.
template <int FOLD> __device__ __forceinline__ void load_staged(uint32_t (&b)[16], Pairs<FOLD>& p, const __half* x, const float2* e, const float2* o) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(x + 32 * h));
        b[4 * h] = u.x; b[4 * h + 1] = u.y; b[4 * h + 2] = u.z; b[4 * h + 3] = u.w;
    }
#pragma unroll
    for (int f = 0; f < 128 / FOLD; ++f) { p.v[f][0] = __ldg(e + f); p.v[f][1] = __ldg(o + f); }
}
// What a warp has of a staged unit (stage_unit below).
template <class X, int FOLD> __device__ __forceinline__ void stage_values(float (&v)[4], __half* out, float2* pair, int lane) {
    float2 s = make_float2(1.f, 1.f);
    if constexpr (Elem<X>::code != VELA_T_F16) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
        s = row_scale(__reduce_max_sync(0xffffffffu, top));
    }
    const uint32_t lo = half2_bits(v[0] * s.x, v[1] * s.x), hi = half2_bits(v[2] * s.x, v[3] * s.x);
    *reinterpret_cast<uint2*>(out + 4 * lane) = make_uint2(lo, hi);
    const float2 fl = __half22float2(*reinterpret_cast<const __half2*>(&lo)), fh = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    float sum = (fl.x + fl.y) + (fh.x + fh.y);
#pragma unroll
    for (int o = 1; o < FOLD / 4; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane % (FOLD / 4) == 0) pair[lane / (FOLD / 4)] = make_float2(s.y, sum);
}
// Stages one unit of a row of X, a warp together: columns 4 lane .. 4 lane + 3 (n of them exist, from p on) to `out` (the unit's
// 128 values); the first lane of each fold writes its pair {factor that the staged values have lost, their sum}.
template <class X, int FOLD> __device__ __forceinline__ void stage_unit(const X* p, int n, __half* out, float2* pair, int lane) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? Elem<X>::get(p[i]) : 0.f;
    stage_values<X, FOLD>(v, out, pair, lane);
}
// One unit of a row of floats (x as above) as the sum of two f16 values.  Plain loads: another block of the same kernel may have
// written them.  left is a multiple of 8, p aligned to 16 bytes.
template <int FOLD> __device__ __forceinline__ void load_floats(uint32_t (&b)[32], Pairs<FOLD>& p, const float* x, int left, int t) {
    float v[32];
    uint32_t top = 0;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
        if (left > 32 * h) { lo = *reinterpret_cast<const float4*>(x + 32 * h); hi = *reinterpret_cast<const float4*>(x + 32 * h + 4); }
        v[8 * h] = lo.x; v[8 * h + 1] = lo.y; v[8 * h + 2] = lo.z; v[8 * h + 3] = lo.w;
        v[8 * h + 4] = hi.x; v[8 * h + 5] = hi.y; v[8 * h + 6] = hi.z; v[8 * h + 7] = hi.w;
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    const float2 s = row_scale(top);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float v0 = v[2 * i] * s.x, v1 = v[2 * i + 1] * s.x;
        b[i] = half2_bits(v0, v1);
        const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&b[i]));
        b[16 + i] = half2_bits(v0 - r.x, v1 - r.y);
    }
    make_pairs<FOLD>(p, b, t, s.y);
}

// The products of one unit, scaled and added to acc: c0, c1 = row g of the weights and columns 2t, 2t + 1; c2, c3 = row g + 8.
template <Kind KIND, int FOLD, bool ZERO>
__device__ __forceinline__ void multiply(float (&acc)[4], const Unit<FOLD, ZERO>& W, const uint32_t (&b)[regs<KIND>()], const Pairs<FOLD>& p, bool f16) {
    constexpr int HALVES = FOLD / 32;
    const uint32_t u[8] = {W.w[0].x, W.w[0].y, W.w[0].z, W.w[0].w, W.w[1].x, W.w[1].y, W.w[1].z, W.w[1].w};
#pragma unroll
    for (int f = 0; f < 128 / FOLD; ++f) {
        float d[4] = {};
#pragma unroll
        for (int h = f * HALVES; h < (f + 1) * HALVES; ++h)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t v = u[2 * h + j], v8 = v >> 8;
                const uint32_t a[4] = {v & 0x000f000fu, v & 0x00f000f0u, v8 & 0x000f000fu, v8 & 0x00f000f0u};
                if constexpr (KIND == H) Ops<__half>::mma(d, a, b[16 + 4 * h + 2 * j], b[16 + 4 * h + 2 * j + 1]);
                Ops<__half>::mma(d, a, b[4 * h + 2 * j], b[4 * h + 2 * j + 1]);
            }
        const float2 s = scale_pair(W.s[f], f16);
        const float z0 = ZERO ? float(W.z[ZERO ? f : 0] & 0xffu) : 8.f, z1 = ZERO ? float(W.z[ZERO ? f : 0] >> 8) : 8.f;
        const float2 e = p.v[f][0], o = p.v[f][1];
        acc[0] = fmaf(s.x * e.x, fmaf(0x1p24f, d[0], -z0 * e.y), acc[0]);
        acc[1] = fmaf(s.x * o.x, fmaf(0x1p24f, d[1], -z0 * o.y), acc[1]);
        acc[2] = fmaf(s.y * e.x, fmaf(0x1p20f, d[2], -z1 * e.y), acc[2]);
        acc[3] = fmaf(s.y * o.x, fmaf(0x1p20f, d[3], -z1 * o.y), acc[3]);
    }
}

// ---------------------------------------------------------------- streaming row tiles past stationary activations
constexpr int COL = 20;                   // floats from one column's 16 sums to the next: stores are free of bank conflicts
__host__ __device__ constexpr size_t sum_bytes(int cols, int rounds) { return size_t(WARPS) * cols * COL * 4 * rounds; }

// The block's share: row tiles r0 .. r1 - 1 (at least one) of a matrix whose first row tile is number tile0, against `cols` <= 8
// activation rows.  Weights are loaded one round ahead.  A warp's sums go to shared memory and are added there, in the order of the
// warps, once for `room` rounds (sum_bytes).  load(u, b, pairs): operands of unit u, by a whole warp; out(rt, col, row or half row,
// sums): called by one thread for each row of 16, or with PAIRED for each i < 8 with the sums of rows i and i + 8.
template <Kind KIND, int UW, int FOLD, bool ZERO, bool PAIRED, class LOAD, class OUT>
__device__ __forceinline__ void stream(const Weights& W, size_t tile0, int r0, int r1, int cols, const Split& split, float* sums, int room, LOAD load, OUT out) {
    typedef Unit<FOLD, ZERO> U;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int nu = units(W), nrow = r1 - r0, per = 7 - W.gshift;
    const int ks = split.ks, slots = split.slots, chunks = split.chunks, sl = quot(warp, ks), kw = warp - sl * ks;
    const int total = quot(max(nrow - sl + slots - 1, 0), slots);      // of this warp, if it has a slot
    const int rounds = quot(nrow + slots - 1, slots), most = min(rounds, room);
    float* const mine = sums + size_t(warp) * most * cols * COL;
    auto count = [&](int base, int n) { return sl < slots ? max(0, min(n, total - base)) : 0; };      // rounds with a row tile for this warp

    // Where the next round to be loaded lies, for a chunk's UW units.  Units beyond the last are the last one again, and so are the
    // second tile and the groups that the last unit may lack: they meet activations of zero.
    const uint4* fq = nullptr;
    const uint32_t* fs = nullptr;
    const uint16_t* fz = nullptr;
    int o0[UW], o1[UW], so[UW][128 / FOLD];
    const int qstep = slots * W.kt * 32, sstep = slots * W.ng * 8;
    auto seek = [&](int base, int c) {
        const int u0 = (c * ks + kw) * UW, uc = min(u0, nu - 1);
        const size_t tile = tile0 + r0 + base * slots + sl;
        fq = W.q + (tile * W.kt + 2 * size_t(uc)) * 32 + lane;
        fs = W.scale + (tile * W.ng + (size_t(uc) << per)) * 8 + g;
        if constexpr (ZERO) fz = W.zero + (tile * W.ng + (size_t(uc) << per)) * 8 + g;
#pragma unroll
        for (int i = 0; i < UW; ++i) {
            const int u = min(u0 + i, nu - 1);
            o0[i] = (u - uc) * 64;
            o1[i] = o0[i] + (2 * u + 1 < W.kt ? 32 : 0);
#pragma unroll
            for (int f = 0; f < 128 / FOLD; ++f) so[i][f] = (((u - uc) << per) + min((f * FOLD) >> W.gshift, W.ng - 1 - (u << per))) * 8;
        }
    };
    auto fetch = [&](U (&s)[UW]) {
#pragma unroll
        for (int i = 0; i < UW; ++i) {
            s[i].w[0] = load_tile(fq + o0[i]);
            s[i].w[1] = load_tile(fq + o1[i]);
#pragma unroll
            for (int f = 0; f < 128 / FOLD; ++f) {
                s[i].s[f] = __ldg(fs + so[i][f]);
                if constexpr (ZERO) s[i].z[f] = __ldg(fz + so[i][f]);
            }
        }
        fq += qstep; fs += sstep;
        if constexpr (ZERO) fz += sstep;
    };
    uint32_t b[UW][regs<KIND>()];
    Pairs<FOLD> p[UW];
    U one[UW], two[UW];
    seek(0, 0);
    if (count(0, most) > 0) fetch(one);
    for (int base = 0; base < rounds; base += most) {
        const int n = min(most, rounds - base), have = count(base, n);
        for (int c = 0; c < chunks; ++c) {
            if (chunks > 1 || base == 0) {
#pragma unroll
                for (int i = 0; i < UW; ++i) {
                    const int u = (c * ks + kw) * UW + i;
                    load(min(u, nu - 1), b[i], p[i]);
                    if (u >= nu) {
#pragma unroll
                        for (int r = 0; r < regs<KIND>(); ++r) b[i][r] = 0u;
#pragma unroll
                        for (int f = 0; f < 128 / FOLD; ++f) p[i].v[f][0] = p[i].v[f][1] = make_float2(0.f, 0.f);
                    }
                }
            }
            if (c > 0 || base > 0) {                        // what was fetched at the end of the last chunk
#pragma unroll
                for (int i = 0; i < UW; ++i) one[i] = two[i];
            }
            float* d = mine + 2 * t * COL + g;
            auto work = [&](const U (&w)[UW]) {
                float acc[4] = {};
#pragma unroll
                for (int i = 0; i < UW; ++i) multiply<KIND, FOLD, ZERO>(acc, w[i], b[i], p[i], W.f16);
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (2 * t + i < cols) {
                        float* q = d + i * COL;
                        if (c) { acc[i] += q[0]; acc[i + 2] += q[8]; }
                        q[0] = acc[i]; q[8] = acc[i + 2];
                    }
                d += cols * COL;
            };
            int j = 0;
            for (; j + 2 < have; j += 2) {
                fetch(two); work(one);
                fetch(one); work(two);
            }
            if (j + 1 < have) {
                fetch(two); work(one);
#pragma unroll
                for (int i = 0; i < UW; ++i) one[i] = two[i];
                ++j;
            }
            const bool wrap = c + 1 == chunks;
            if (!wrap || base + n < rounds) {
                seek(wrap ? base + n : base, wrap ? 0 : c + 1);
                if (wrap ? count(base + n, min(most, rounds - base - n)) > 0 : have > 0) fetch(two);
            }
            if (j < have) work(one);
        }
        __syncthreads();
        constexpr int ROWS = PAIRED ? 8 : 16;
        // thread i sums row i mod ROWS of every WARPS * 32 / ROWS-th column of a row tile
        const int row = threadIdx.x % ROWS;
        for (int i = threadIdx.x / ROWS; i < n * slots * cols; i += WARPS * 32 / ROWS) {
            const int rr = quot(i, cols), col = i - rr * cols, jj = quot(rr, slots), s = rr - jj * slots, rt = r0 + (base + jj) * slots + s;
            if (rt >= r1) continue;
            const float* e = sums + ((s * ks * most + jj) * cols + col) * COL + row;
            float v = 0.f, w = 0.f;
#pragma unroll 4
            for (int k = 0; k < ks; ++k) { v += e[0]; if (PAIRED) w += e[8]; e += most * cols * COL; }
            out(rt, col, row, v, w);
        }
        __syncthreads();
    }
}

}  // namespace w4
}  // namespace vela
