// The expert layer for very few tokens: every (token, expert) pair by itself, in two plain kernels.  There is next to no weight to
// share between tokens then, and latency is what counts.
//   few_up: the four blocks of a cluster route by themselves (each forms a quarter of the scores on the tensor cores and gives them
//   to the others through their shared memory; all of them then choose), and each takes its items of the gate and up products: an
//   item is one row tile of one pair, ks warps share its columns.  So there is no kernel of its own for routing, nor a wait between
//   it and the products.
//   few_down: an item is one row tile of one token's output; its sum runs over the token's experts and their hidden columns, shared
//   out among the block's warps.  A hidden value is the sum of two bf16 values (16 bits), which are two columns of the same product.
//
// One token, 8 of 64 experts of 2048 x 1024, bf16: 16.3 us a layer, 26 MB; 2 of 16 experts of 1024 x 512: 8.2 us.  Scoring and
// choosing take about 5 us of the first kernel, the rest is latency: the first fetch of weights waits for the choice, and code that
// runs once comes from a cold instruction cache.
#pragma once
#include "w4.cuh"

namespace vela {
namespace few {

constexpr int WARPS = 16, TOKENS = 8, EXPERTS = 128, PAIRS = 32;      // of few_up_kernel; what it can take
constexpr int PART = 9;                   // floats from one expert's 8 partial scores to the next's

constexpr int RANKS = 4;                  // blocks of a cluster, which share the scoring

// Shared memory: the staged rows (halves, then pairs), then this block's part of the scores
template <int FOLD> __host__ __device__ constexpr size_t stage_bytes(int tokens, int nu) { return size_t(tokens) * nu * (256 + 8 * (128 / FOLD)); }
__host__ __device__ constexpr int score_tiles(int E) { return ((E + 15) / 16 + RANKS - 1) / RANKS; }      // of 16 experts, for one block
template <int FOLD> __host__ __device__ constexpr size_t up_bytes(int tokens, int nu, int E) {
    return stage_bytes<FOLD>(tokens, nu) + size_t(WARPS) * score_tiles(E) * 16 * PART * 4;
}

// Scores of up to 8 tokens: this warp's share of the columns, 32 at a time, for the tiles of 16 experts rank, rank + RANKS, ...;
// part[e * PART + token] with e counted within those tiles.  X: bf16 or f16, the router's type too; D % 8 == 0, rows aligned to 16
// bytes.
template <class X> __device__ __forceinline__ void part_scores(const X* x, int ldx, int tn, const X* router, int E, int D, float* part, int rank, int warp, int lane) {
    const int g = lane >> 2, t = lane & 3;
    const X* row = x + size_t(min(g, tn - 1)) * ldx;
    for (int e0 = 16 * rank, at = 0; e0 < E; e0 += 16 * RANKS, at += 16) {
        const X* lo = router + size_t(min(e0 + g, E - 1)) * D;
        const X* hi = router + size_t(min(e0 + g + 8, E - 1)) * D;
        float c[4] = {};
#pragma unroll 4
        for (int k0 = warp * 32; k0 < D; k0 += WARPS * 32) {
            const int k = k0 + 8 * t;
            uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a, v = a;
            if (k < D) {
                a = __ldg(reinterpret_cast<const uint4*>(lo + k)); b = __ldg(reinterpret_cast<const uint4*>(hi + k)); v = __ldg(reinterpret_cast<const uint4*>(row + k));
            }
            const uint32_t p[4] = {a.x, b.x, a.y, b.y}, q[4] = {a.z, b.z, a.w, b.w};
            w4::Ops<X>::mma(c, p, v.x, v.y);
            w4::Ops<X>::mma(c, q, v.z, v.w);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) part[(at + g + 8 * (i >> 1)) * PART + 2 * t + (i & 1)] = c[i];
    }
}

// Adds a unit of one row tile to acc (rows g and g + 8): one activation row, staged in shared memory (w4_stream.cuh: stage_unit).
// x: column 8 t of the unit.
template <int FOLD, bool ZERO>
__device__ __forceinline__ void one_staged(float (&acc)[2], const w4::Unit<FOLD, ZERO>& W, const __half* x, const float2* pair, bool f16) {
    constexpr int HALVES = FOLD / 32;
#pragma unroll
    for (int f = 0; f < 128 / FOLD; ++f) {
        float c[4] = {}, d[4] = {};                // two chains: a product waits for the one before it in its chain
#pragma unroll
        for (int h = f * HALVES; h < (f + 1) * HALVES; ++h) {
            const uint4 b = *reinterpret_cast<const uint4*>(x + 32 * h);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint4 w = W.w[h >> 1];
                const uint32_t v = h & 1 ? (j ? w.w : w.z) : (j ? w.y : w.x), v8 = v >> 8;
                const uint32_t a[4] = {v & 0x000f000fu, v & 0x00f000f0u, v8 & 0x000f000fu, v8 & 0x00f000f0u};
                w4::Ops<__half>::mma(j ? d : c, a, j ? b.z : b.x, j ? b.w : b.y);
            }
        }
        const float2 s = w4::scale_pair(W.s[f], f16), p = pair[f];
        const float z0 = ZERO ? float(W.z[ZERO ? f : 0] & 0xffu) : 8.f, z1 = ZERO ? float(W.z[ZERO ? f : 0] >> 8) : 8.f;
        acc[0] = fmaf(s.x * p.x, fmaf(0x1p24f, c[0] + d[0], -z0 * p.y), acc[0]);
        acc[1] = fmaf(s.y * p.x, fmaf(0x1p20f, c[2] + d[2], -z1 * p.y), acc[1]);
    }
}

}  // namespace few
}  // namespace vela
