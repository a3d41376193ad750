// A mixture-of-experts layer for a few tokens on 4-bit weights, in two kernels, of two forms.  What bounds the layer is the reading
// of the chosen experts' weights; with one or two tokens it is latency.
//
// Very few tokens (moe_few.cuh): few_up_kernel routes and does the gate and up products, few_down_kernel the down products and
// their weighed sums.
//
// Else: route_kernel, a cluster of 8 blocks for each token, scores the experts (a warp for each), chooses, and stages the token's
// row for the products (w4_stream.cuh); it also clears the other kernel's counters.  expert_kernel, one block on each SM (a
// cooperative launch), does all chosen experts' gate and up products, then their down products, then the weighed sums, with a
// barrier over the whole grid in between.  An item is one row tile of one expert, for all tokens that chose it (columns of one
// product, so weights are read once for every 8 of them); a block takes a run of neighbouring items, so an expert's activations
// stay in its registers.  A barrier costs about 1.5 us, over which the next weights are already on their way to the L2 cache.
//   Up: a row tile is 8 gate rows and their 8 up rows, so one thread sums both parts of a hidden value, which is kept as a float.
//   Down: the result of each token and expert by itself, as floats; then each output is summed over the token's experts in the
//   order of their places.
// 32 tokens, 4 of 32 experts of 4096 x 1536, bf16: 101 to 103 us for 308 MB, 46 % of what a copy reaches.  Routing and the gap to
// the next kernel take 10 us; blocks end up to 12 us apart in each phase (their shares are equal, their bandwidth is not; handing out
// the last items as blocks get free costs more, since every run begins anew), and the down phase has a chain of 16 dependent products
// for each unit.
#include "host_util.h"
#include "tc.cuh"
#include "moe_few.cuh"
#include "w4_stream.cuh"
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cooperative_groups.h>

namespace vela {
namespace {
namespace cg = cooperative_groups;

constexpr int E_MAX = 1024, K_MAX = 32;
constexpr int T_BLOCK = 32;               // tokens of one expert_kernel launch
constexpr int RANKS = 8, ROUTE_WARPS = 8; // of route_kernel
constexpr int WARPS = w4::WARPS;          // of expert_kernel
constexpr int FEW_SMEM = 96 * 1024;           // of two blocks on an SM
constexpr size_t FEW_ROUTER = 512 * 1024;     // elements of the router that a cluster reads
constexpr int COUNTERS = 2;               // one for each barrier
constexpr size_t ROOM_BYTES = w4::sum_bytes(1, w4::ROOM);
static __device__ unsigned g_moe_err;

struct MoeArgs {
    w4::Weights up, down;             // expert 0's; the others follow
    const void* X; const void* router; const float* bias; void* Y;
    int32_t* ids; float* weights;     // [T][topk], the caller's or the workspace's
    __half* xs; float2* xp;           // staged rows [T][units of D], their pairs
    __nv_bfloat16* hi; __nv_bfloat16* lo;     // few tokens: hidden values [T * topk][units of I]
    float* h; float* o;               // hidden values [T_BLOCK * topk][I], experts' results [T_BLOCK * topk][D rounded up to 16]
    unsigned* count;                  // [launch][COUNTERS]
    int D, I, E, topk, T, ldx, ldy, score, renorm, ytype;
    float scale;
    bool vecx, vecr;
    int t0, tn;                       // expert_kernel: its tokens
    w4::Split split_up, split_down;
    unsigned* err; long long limit; unsigned extra;
};

// a token's row times a router row, by one warp, with 8 loads of each in flight
template <class X, class RW> __device__ __forceinline__ float dot_row(const X* x, const RW* w, int D, bool vecx, bool vecr, int lane) {
    float s[4] = {};
    if (vecx && vecr) {                               // D % 8 == 0
        for (int k0 = 8 * lane; k0 < D; k0 += 8 * 256) {
            uint4 a[8][sizeof(X) / 2], b[8][sizeof(RW) / 2];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int k = min(k0 + 256 * j, D - 8);
#pragma unroll
                for (int i = 0; i < int(sizeof(RW) / 2); ++i) b[j][i] = __ldg(reinterpret_cast<const uint4*>(w + k) + i);
#pragma unroll
                for (int i = 0; i < int(sizeof(X) / 2); ++i) a[j][i] = __ldg(reinterpret_cast<const uint4*>(x + k) + i);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (k0 + 256 * j >= D) break;
                const X* u = reinterpret_cast<const X*>(a[j]);
                const RW* v = reinterpret_cast<const RW*>(b[j]);
#pragma unroll
                for (int i = 0; i < 8; ++i) s[j & 3] = fmaf(Elem<X>::get(u[i]), Elem<RW>::get(v[i]), s[j & 3]);
            }
        }
    } else {
        for (int k = 8 * lane; k < D; k += 256) {
            float a[8], b[8];
            load8(w + k, min(8, D - k), vecr, b);
            load8(x + k, min(8, D - k), vecx, a);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[0] = fmaf(a[i], b[i], s[0]);
        }
    }
    float v = (s[0] + s[1]) + (s[2] + s[3]);
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// order-preserving bits of a float that is not a NaN; both zeros alike
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __float_as_uint(v + 0.f);
    return u >> 31 ? ~u : u | 0x80000000u;
}

// What the choice goes by: the larger key first.  Without a selection bias that is the score, whose order the probabilities have
// too, but not in 32 bits where several are 0 (softmax: 104 below the largest score) or 1 (sigmoid: from 17 on).  A NaN comes last,
// after experts that a selection bias of minus infinity masks; 0 is left for places beyond the last expert.
__device__ __forceinline__ uint32_t choice_key(float prob, float score, const float* bias, int e) {
    const float w = bias ? prob + __ldg(bias + e) : score;
    return w != w ? 1u : ordered(w);
}

// an expert's share of the softmax's sum: none where the score is a NaN, so that one such expert does not spoil the others'
// probabilities
__device__ __forceinline__ float soft_term(float z, float most) { return z != z ? 0.f : expf(z - most); }

// Weight of a token's j-th choice: its probability p[j], with `renorm` divided by the sum over the choices.  A sum below 1e-30 has
// probabilities in it that have lost their bits or are 0; to 30 digits they are exp(score) then (sigmoid) or a multiple of it
// (softmax), so the scores z give the quotients, taken from the largest one on.
__device__ __forceinline__ float weight(const float* p, const float* z, int topk, int j, const MoeArgs& a) {
    if (!a.renorm) return p[j] * a.scale;
    float s = 0.f;
    for (int i = 0; i < topk; ++i) s += p[i];
    if (s < 1e-30f) {
        float most = z[0];
        for (int i = 1; i < topk; ++i) most = fmaxf(most, z[i]);
        s = 0.f;
        for (int i = 0; i < topk; ++i) s += expf(z[i] - most);
        return expf(z[j] - most) / s * a.scale;
    }
    return p[j] / s * a.scale;
}

template <class X, class RW, int FOLD> __global__ void __cluster_dims__(RANKS, 1, 1) __launch_bounds__(ROUTE_WARPS * 32) route_kernel(const MoeArgs a) {
    __shared__ float p[E_MAX], prob[E_MAX], top[K_MAX], topz[K_MAX];
    __shared__ __align__(16) uint32_t key[E_MAX];
    const int E4 = (a.E + 3) & ~3;
    cg::cluster_group cluster = cg::this_cluster();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tok = blockIdx.y, rank = blockIdx.x;
    const int gw = rank * ROUTE_WARPS + warp;
    const X* x = static_cast<const X*>(a.X) + size_t(tok) * a.ldx;
    float* lead = cluster.map_shared_rank(p, 0);
    cluster.sync();                                        // all have begun: their shared memory may be written
    for (int e = gw; e < a.E; e += RANKS * ROUTE_WARPS) {
        const float s = dot_row(x, static_cast<const RW*>(a.router) + size_t(e) * a.D, a.D, a.vecx, a.vecr, lane);
        if (lane == 0) lead[e] = s;
    }
    cluster.sync();
    if (rank != 0) {
        // the others: the staged row and the counters
        const int i = gw - ROUTE_WARPS, n = (RANKS - 1) * ROUTE_WARPS, nu = w4::units(a.up);
        for (int u = i; u < nu; u += n)
            w4::stage_unit<X, FOLD>(x + u * 128 + 4 * lane, a.D - u * 128 - 4 * lane, a.xs + (size_t(tok) * nu + u) * 128, a.xp + (size_t(tok) * nu + u) * (128 / FOLD), lane);
        if (tok % T_BLOCK == 0 && i == 0 && lane < COUNTERS) a.count[tok / T_BLOCK * COUNTERS + lane] = 0;
        return;
    }
    // Every warp forms the softmax's maximum and sum for itself, in the same order.
    float m = -INFINITY, sum = 0.f;
    if (a.score == 0) {
        for (int e = lane; e < a.E; e += 32) m = fmaxf(m, p[e]);
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        for (int e = lane; e < a.E; e += 32) sum += soft_term(p[e], m);
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    for (int e = threadIdx.x; e < E4; e += ROUTE_WARPS * 32) {
        uint32_t v = 0;                                    // below every expert's
        if (e < a.E) {
            const float q = a.score == 0 ? expf(p[e] - m) / sum : 1.f / (1.f + expf(-p[e]));
            prob[e] = q;
            v = choice_key(q, p[e], a.bias, e);
        }
        key[e] = v;
    }
    __syncthreads();
    // An expert's place is the number of those before it: larger ones, and equal ones of lower number.
    for (int e = threadIdx.x; e < a.E; e += ROUTE_WARPS * 32) {
        const uint32_t v = key[e];
        int r = 0;
        for (int o = 0; o < E4; o += 4) {
            const uint4 k = *reinterpret_cast<const uint4*>(key + o);
            r += (k.x > v || (k.x == v && o < e)) + (k.y > v || (k.y == v && o + 1 < e)) + (k.z > v || (k.z == v && o + 2 < e)) + (k.w > v || (k.w == v && o + 3 < e));
        }
        if (r < a.topk) { top[r] = prob[e]; topz[r] = p[e]; a.ids[size_t(tok) * a.topk + r] = e; }
    }
    __syncthreads();
    if (int(threadIdx.x) < a.topk) a.weights[size_t(tok) * a.topk + threadIdx.x] = weight(top, topz, a.topk, threadIdx.x, a);
}

template <class X, int FOLD, bool ZERO> __global__ void __cluster_dims__(few::RANKS, 1, 1) __launch_bounds__(few::WARPS * 32, 2) few_up_kernel(const MoeArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float s_z[few::TOKENS][few::EXPERTS], s_p[few::TOKENS][few::EXPERTS], s_top[few::PAIRS], s_topz[few::PAIRS];
    __shared__ __align__(16) uint32_t s_key[few::TOKENS][few::EXPERTS];
    __shared__ int32_t s_ids[few::PAIRS];
    __shared__ float s_sum[few::WARPS][16];
    asm volatile("griddepcontrol.launch_dependents;");     // few_down_kernel may be brought up
    cg::cluster_group cluster = cg::this_cluster();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = lane & 3, nu = w4::units(a.up), rank = blockIdx.x % few::RANKS;
    const X* x = static_cast<const X*>(a.X);
    __half* xs = reinterpret_cast<__half*>(smem);
    float2* xp = reinterpret_cast<float2*>(smem + size_t(a.T) * nu * 256);
    float* part = reinterpret_cast<float*>(smem + few::stage_bytes<FOLD>(a.T, nu));
    const int mine = few::score_tiles(a.E) * 16;          // experts whose scores this block forms, at most
    few::part_scores<X>(x, a.ldx, a.T, static_cast<const X*>(a.router), a.E, a.D, part + warp * mine * few::PART, rank, warp, lane);
    for (int i0 = warp; i0 < a.T * nu; i0 += 4 * few::WARPS) {     // four units under way at a time
        uint2 raw[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = i0 + j * few::WARPS, tok = w4::quot(i, nu), c = (i - tok * nu) * 128 + 4 * lane;
            raw[j] = i < a.T * nu && c < a.D ? __ldg(reinterpret_cast<const uint2*>(x + size_t(tok) * a.ldx + c)) : make_uint2(0u, 0u);      // D % 8 == 0
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = i0 + j * few::WARPS;
            if (i >= a.T * nu) break;
            const X* e = reinterpret_cast<const X*>(&raw[j]);
            float v[4] = {Elem<X>::get(e[0]), Elem<X>::get(e[1]), Elem<X>::get(e[2]), Elem<X>::get(e[3])};
            w4::stage_values<X, FOLD>(v, xs + size_t(i) * 128, xp + size_t(i) * (128 / FOLD), lane);
        }
    }
    __syncthreads();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");       // all have begun: their shared memory may be written
    for (int i = threadIdx.x; i < mine * few::TOKENS; i += few::WARPS * 32) {
        const int at = i >> 3, tok = i & 7, e = (at / 16 * few::RANKS + rank) * 16 + at % 16;
        if (e >= a.E || tok >= a.T) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < few::WARPS; ++w) v += part[(w * mine + at) * few::PART + tok];
        for (int r = 0; r < few::RANKS; ++r) cluster.map_shared_rank(&s_z[0][0], r)[tok * few::EXPERTS + e] = v;
    }
    cluster.sync();
    // probabilities and keys: a warp for each token
    const int E4 = (a.E + 3) & ~3;
    if (warp < a.T) {
        const float* z = s_z[warp];
        float m = -INFINITY, sum = 0.f;
        if (a.score == 0) {
            for (int e = lane; e < a.E; e += 32) m = fmaxf(m, z[e]);
            for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            for (int e = lane; e < a.E; e += 32) sum += soft_term(z[e], m);
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        for (int e = lane; e < E4; e += 32) {
            uint32_t v = 0;                                // below every expert's
            if (e < a.E) {
                const float q = a.score == 0 ? expf(z[e] - m) / sum : 1.f / (1.f + expf(-z[e]));
                s_p[warp][e] = q;
                v = choice_key(q, z[e], a.bias, e);
            }
            s_key[warp][e] = v;
        }
    }
    __syncthreads();
    // an expert's place is the number of those before it: larger ones, and equal ones of lower number
    for (int i = threadIdx.x; i < a.T * few::EXPERTS; i += few::WARPS * 32) {
        const int tok = i / few::EXPERTS, e = i % few::EXPERTS;
        if (e >= a.E) continue;
        const uint32_t v = s_key[tok][e];
        int r = 0;
#pragma unroll 1
        for (int o = 0; o < E4; o += 4) {
            const uint4 k = *reinterpret_cast<const uint4*>(&s_key[tok][o]);
            r += (k.x > v || (k.x == v && o < e)) + (k.y > v || (k.y == v && o + 1 < e)) + (k.z > v || (k.z == v && o + 2 < e)) + (k.w > v || (k.w == v && o + 3 < e));
        }
        if (r < a.topk) { s_ids[tok * a.topk + r] = e; s_top[tok * a.topk + r] = s_p[tok][e]; s_topz[tok * a.topk + r] = s_z[tok][e]; }
    }
    __syncthreads();
    // The last block's last warp writes the choice: it is the one that is left without an item unless they come out even.
    if (blockIdx.x == gridDim.x - 1 && warp == few::WARPS - 1 && lane < a.T * a.topk) {
        static_assert(few::PAIRS <= 32, "a lane for each pair");
        const int at = w4::quot(lane, a.topk) * a.topk;
        a.ids[lane] = s_ids[lane];
        a.weights[lane] = weight(s_top + at, s_topz + at, a.topk, lane - at, a);
    }
    // the hidden rows' padding
    const int wide = w4::units(a.down) * 128, P = a.T * a.topk;
    for (int p = blockIdx.x; p < P; p += gridDim.x)
        for (int c = a.I + threadIdx.x; c < wide; c += few::WARPS * 32) { a.hi[size_t(p) * wide + c] = __nv_bfloat16(0.f); a.lo[size_t(p) * wide + c] = __nv_bfloat16(0.f); }
    const int rt = w4::row_tiles(a.up), items = P * rt, ks = a.split_up.ks, slots = a.split_up.slots, sl = w4::quot(warp, ks), kw = warp - sl * ks;
    for (int base = blockIdx.x; base < items; base += gridDim.x * slots) {
        const int it = base + gridDim.x * sl;
        float acc[2] = {};
        const int p = w4::quot(min(it, items - 1), rt), r = it - p * rt;
        if (sl < slots && it < items) {
            const size_t tile = size_t(s_ids[p]) * rt + r;
            const __half* row = xs + size_t(w4::quot(p, a.topk)) * nu * 128 + 8 * t;
            const float2* pair = xp + size_t(w4::quot(p, a.topk)) * nu * (128 / FOLD);
            constexpr int U = 2;                           // units under way at a time
            w4::RowPtr at = w4::row_ptr(a.up, tile, kw, lane);
            if (kw == 0 && lane == 0) w4::prefetch_l2(at.q, a.up.kt * 512);
#pragma unroll 1
            for (int u = kw; u < nu; u += U * ks) {
                w4::Unit<FOLD, ZERO> w[U];
#pragma unroll
                for (int i = 0; i < U; ++i)
                    if (u + i * ks < nu) { w4::load_last(w[i], at, a.up, u + i * ks); w4::advance(at, a.up, ks); }
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const int v = u + i * ks;
                    if (v < nu) few::one_staged<FOLD, ZERO>(acc, w[i], row + v * 128, pair + v * (128 / FOLD), a.up.f16);
                }
            }
        }
        if (t == 0) { s_sum[warp][lane >> 2] = acc[0]; s_sum[warp][8 + (lane >> 2)] = acc[1]; }
        __syncthreads();
        if (kw == 0 && sl < slots && lane < 8 && it < items) {
            float gate = 0.f, up = 0.f;
            for (int w = 0; w < ks; ++w) { gate += s_sum[warp + w][lane]; up += s_sum[warp + w][8 + lane]; }
            const float h = gate / (1.f + expf(-gate)) * up;
            const __nv_bfloat16 hi = __float2bfloat16_rn(h);
            const float hf = __bfloat162float(hi);
            const size_t at = size_t(p) * wide + r * 8 + lane;
            a.hi[at] = hi;
            a.lo[at] = __float2bfloat16_rn(isinf(hf) ? 0.f : h - hf);
        }
        __syncthreads();
    }
}

template <int FOLD, bool ZERO, int WARPS> __global__ void __launch_bounds__(WARPS * 32, 32 / WARPS) few_down_kernel(const MoeArgs a) {
    __shared__ float s_sum[WARPS][16];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int rt = w4::row_tiles(a.down), nu = w4::units(a.down), items = a.T * rt, n = a.topk * nu, wide = nu * 128;
    const w4::Consts k = w4::consts<__nv_bfloat16>();
    // few_up_kernel has ended and its results are visible; they were written while this kernel was already there, so all are read
    // by plain loads
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // the two terms of a hidden value are columns 0 and 1 of the product (and 2 to 7 again, which are not used)
    const __nv_bfloat16* h = (g & 1 ? a.lo : a.hi) + 8 * t;
    for (int it = blockIdx.x; it < items; it += gridDim.x) {
        const int tok = w4::quot(it, rt), r = it - tok * rt;
        float acc[2] = {};
#pragma unroll 1
        for (int q = warp; q < n; q += WARPS) {
            const int j = w4::quot(q, nu), u = q - j * nu, p = tok * a.topk + j;
            w4::Unit<FOLD, ZERO> w[1];
            w4::load_last(w[0], w4::row_ptr(a.down, size_t(a.ids[p]) * rt + r, u, lane), a.down, u);
            float c[1][1][4] = {};
            const __nv_bfloat16* x[1] = {h + size_t(p) * wide + u * 128};
            w4::unit<VELA_T_BF16, true, 1, 1, false>(c, w, x, 0, a.down.f16, k, [](int, int) { return make_float2(1.f, 1.f); });
            const float y = a.weights[p];
            acc[0] = fmaf(y, c[0][0][0] + c[0][0][1], acc[0]);
            acc[1] = fmaf(y, c[0][0][2] + c[0][0][3], acc[1]);
        }
        if (t == 0) { s_sum[warp][g] = acc[0]; s_sum[warp][8 + g] = acc[1]; }
        __syncthreads();
        const int col = r * 16 + threadIdx.x;
        if (threadIdx.x < 16 && col < a.D) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) v += s_sum[w][threadIdx.x];
            const size_t at = size_t(tok) * a.ldy + col;
            if (a.ytype == VELA_T_BF16) static_cast<__nv_bfloat16*>(a.Y)[at] = __float2bfloat16_rn(v);
            else static_cast<__half*>(a.Y)[at] = __float2half_rn(v);
        }
        __syncthreads();
    }
}

// Waits until all blocks of the grid have come here; false (and the error word set) if they have not within the limit.
__device__ __forceinline__ bool grid_barrier(unsigned* count, unsigned want, unsigned* err, long long limit, int* flag) {
    __syncthreads();
    if (threadIdx.x == 0) {
        *flag = 1;
        asm volatile("red.release.gpu.global.add.u32 [%0], 1;" :: "l"(count) : "memory");
        const long long t0 = clock64();
        while (true) {
            unsigned seen;
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(count) : "memory");
            if (seen >= want) break;
            if (clock64() - t0 > limit) { atomicCAS(err, 0u, unsigned(DEVERR_TIMEOUT_OTHER)); *flag = 0; break; }
        }
    }
    __syncthreads();
    return *flag != 0;
}

template <int FOLD, bool ZERO> __global__ void __launch_bounds__(WARPS * 32, 1) expert_kernel(const MoeArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int s_n, s_flag;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int grid = gridDim.x, P = a.tn * a.topk, p0 = a.t0 * a.topk;
    float* sums = reinterpret_cast<float*>(smem);
    int32_t* s_list = reinterpret_cast<int32_t*>(smem + ROOM_BYTES);
    int32_t* s_ids = s_list + P;
    int32_t* s_expert = s_ids + P;                  // slot v has expert s_expert[v] and the pairs (token * topk + place) s_at[s_first[v]] .. s_at[s_first[v + 1] - 1], 8 at most
    int32_t* s_first = s_expert + P;
    int32_t* s_cnt = s_first + P + 1;
    int32_t* s_at = s_cnt + a.E;
    int32_t* s_tok = s_at + P;                      // their tokens
    if (warp == 0) {
        for (int e = lane; e < a.E; e += 32) s_cnt[e] = 0;
        __syncwarp();
        for (int i0 = 0; i0 < P; i0 += 32) {           // each pair's place among its expert's, in the order of the pairs
            const int i = i0 + lane, e = i < P ? a.ids[p0 + i] : -1 - lane;
            const unsigned same = __match_any_sync(0xffffffffu, e);
            const int before = __popc(same & ((1u << lane) - 1));
            if (i < P) { s_ids[i] = e; s_list[i] = s_cnt[e] + before; }
            __syncwarp();
            if (i < P && before == 0) s_cnt[e] += __popc(same);
            __syncwarp();
        }
        int n = 0, at = 0;                              // first places and slots, by expert; s_cnt becomes the first place
        for (int e0 = 0; e0 < a.E; e0 += 32) {
            const int e = e0 + lane, c = e < a.E ? s_cnt[e] : 0, v = (c + 7) >> 3;
            if (__ballot_sync(0xffffffffu, c) == 0) continue;
            int ci = c, vi = v;
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, ci, o), y = __shfl_up_sync(0xffffffffu, vi, o);
                if (lane >= o) { ci += x; vi += y; }
            }
            for (int i = 0; i < v; ++i) { s_expert[n + vi - v + i] = e; s_first[n + vi - v + i] = at + ci - c + 8 * i; }
            if (c) s_cnt[e] = at + ci - c;
            n += __shfl_sync(0xffffffffu, vi, 31);
            at += __shfl_sync(0xffffffffu, ci, 31);
        }
        if (lane == 0) { s_n = n; s_first[n] = at; }
        __syncwarp();
        for (int i0 = 0; i0 < P; i0 += 32) { const int i = i0 + lane; if (i < P) { const int q = s_cnt[s_ids[i]] + s_list[i]; s_at[q] = i; s_tok[q] = w4::quot(i, a.topk); } }
    }
    __syncthreads();
    const int V = s_n;
    // Runs of items: this block's row tiles of one slot after another.  ask: a run's weights on their way to the L2 cache, 64 KB of
    // them at most
    auto ask = [&](const w4::Weights& W, int it, int hi) {
        if (threadIdx.x == 0 && it < hi) {
            const int rt = w4::row_tiles(W), v = w4::quot(it, rt), n = min(min(hi - it, rt - (it - v * rt)), max(1, 65536 / (W.kt * 512)));
            w4::prefetch_l2(W.q + (size_t(s_expert[v]) * rt + (it - v * rt)) * W.kt * 32, min(n * W.kt * 512, 65536));
        }
    };
    // the first of the V * rt items that are block b's
    auto share = [&](int rt, int b) { const int q = w4::quot(V * rt, grid); return q * b + min(b, V * rt - q * grid); };
    auto runs = [&](const w4::Weights& W, auto run) {
        const int rt = w4::row_tiles(W);
        const int lo = share(rt, blockIdx.x), hi = share(rt, blockIdx.x + 1);
        for (int it = lo; it < hi;) {
            const int v = w4::quot(it, rt), r0 = it - v * rt, n = min(rt - r0, hi - it);
            it += n;
            ask(W, it, hi);
            run(v, size_t(s_expert[v]) * rt, r0, r0 + n, s_first[v + 1] - s_first[v]);
        }
    };
    auto pair_of = [&](int v, int col) { return s_at[s_first[v] + col]; };

    ask(a.up, share(w4::row_tiles(a.up), blockIdx.x), share(w4::row_tiles(a.up), blockIdx.x + 1));
    runs(a.up, [&](int v, size_t tile0, int r0, int r1, int c) {
        const int nu = w4::units(a.up), room = w4::quot(w4::ROOM, c);
        w4::stream<w4::F, w4::up_units(FOLD), FOLD, ZERO, true>(a.up, tile0, r0, r1, c, a.split_up, sums, room,
            [&](int u, uint32_t (&b)[16], w4::Pairs<FOLD>& p) {
                auto at = [&](int col) { return size_t(a.t0 + s_tok[s_first[v] + min(col, c - 1)]) * nu + u; };     // any row where there is none: its column is not used
                w4::load_staged<FOLD>(b, p, a.xs + at(g) * 128 + 8 * t, a.xp + at(2 * t) * (128 / FOLD), a.xp + at(2 * t + 1) * (128 / FOLD));
            },
            [&](int rt, int col, int i, float gate, float up) { a.h[size_t(pair_of(v, col)) * a.I + rt * 8 + i] = gate / (1.f + expf(-gate)) * up; });
    });
    unsigned* count = a.count + a.t0 / T_BLOCK * COUNTERS;
    ask(a.down, share(w4::row_tiles(a.down), blockIdx.x), share(w4::row_tiles(a.down), blockIdx.x + 1));
    if (!grid_barrier(count, grid + a.extra, a.err, a.limit, &s_flag)) return;

    const int wide = w4::row_tiles(a.down) * 16;
    runs(a.down, [&](int v, size_t tile0, int r0, int r1, int c) {
        w4::stream<w4::H, 1, FOLD, ZERO, false>(a.down, tile0, r0, r1, c, a.split_down, sums, w4::quot(w4::ROOM, c),
            [&](int u, uint32_t (&b)[32], w4::Pairs<FOLD>& p) {
                w4::load_floats<FOLD>(b, p, a.h + size_t(pair_of(v, min(g, c - 1))) * a.I + u * 128 + 8 * t, a.I - u * 128 - 8 * t, t);
            },
            [&](int rt, int col, int row, float y, float) { a.o[size_t(pair_of(v, col)) * wide + rt * 16 + row] = y; });
    });
    if (!grid_barrier(count + 1, grid + a.extra, a.err, a.limit, &s_flag)) return;

    for (int i = blockIdx.x * (WARPS * 32) + threadIdx.x; i < a.tn * a.D; i += grid * (WARPS * 32)) {
        const int tok = w4::quot(i, a.D), n = i - tok * a.D;
        float y = 0.f;
        for (int j = 0; j < a.topk; ++j)
            y = fmaf(__ldg(a.weights + size_t(a.t0 + tok) * a.topk + j), __ldcg(a.o + size_t(tok * a.topk + j) * wide + n), y);
        const size_t at = size_t(a.t0 + tok) * a.ldy + n;
        if (a.ytype == VELA_T_BF16) static_cast<__nv_bfloat16*>(a.Y)[at] = __float2bfloat16_rn(y);
        else static_cast<__half*>(a.Y)[at] = __float2half_rn(y);
    }
}

struct Layout { size_t ids, weights, xs, xp, h, o, hi, lo, count, bytes; };
Layout layout(const vela_moe& L, int T) {
    Layout w;
    const size_t n = size_t(T) * L.topk, nu = (size_t(L.D) + 127) / 128, fold = 128 / L.gate_up.group, some = size_t(std::min(T, T_BLOCK)) * L.topk;
    size_t at = 0;
    auto take = [&](size_t b) { const size_t r = at; at += align_up(b, 256); return r; };
    w.ids = take(n * 4); w.weights = take(n * 4);
    w.xs = take(T * nu * 256); w.xp = take(T * nu * fold * 8);
    w.h = take(some * L.I * 4); w.o = take(some * ((size_t(L.D) + 15) / 16 * 16) * 4);
    // few tokens' rows: small, so always there
    const size_t rows = size_t(few::PAIRS) * ((size_t(L.I) + 127) / 128) * 256;
    w.hi = take(rows); w.lo = take(rows);
    w.count = take((size_t(T) + T_BLOCK - 1) / T_BLOCK * COUNTERS * 4);
    w.bytes = at;
    return w;
}

void check(const vela_moe& L, int T) {
    VELA_REQUIRE(T >= 0 && T <= 65535, "moe_w4: T must lie in 0 .. 65535");
    VELA_REQUIRE(L.D > 0 && L.I > 0 && L.I % 8 == 0 && L.I <= (1 << 20) && L.D <= (1 << 20), "moe_w4: D > 0 and I a positive multiple of 8, 2^20 at most");
    VELA_REQUIRE(L.E > 0 && L.E <= E_MAX && L.topk > 0 && L.topk <= K_MAX && L.topk <= L.E, "moe_w4: E in 1 .. 1024 and topk in 1 .. min(E, 32)");
    VELA_REQUIRE(L.score == 0 || L.score == 1, "moe_w4: score must be 0 (softmax) or 1 (sigmoid)");
    VELA_REQUIRE(L.gate_up.N == 2 * L.I && L.gate_up.K == L.D, "moe_w4: gate_up must be [2 I, D]");
    VELA_REQUIRE(L.down.N == L.D && L.down.K == L.I, "moe_w4: down must be [D, I]");
    VELA_REQUIRE(L.gate_up.group == L.down.group && w4_sizes_ok(16, 16, L.down.group), "moe_w4: gate_up and down need the same group of 32, 64 or 128");
    VELA_REQUIRE((L.gate_up.zero != nullptr) == (L.down.zero != nullptr), "moe_w4: gate_up and down both have zero points or neither");
}

template <int FOLD, bool ZERO> void launch_experts(cudaStream_t st, MoeArgs a) {
    auto* kernel = expert_kernel<FOLD, ZERO>;
    const int grid = sm_count();
    auto run = [&](const w4::Weights& W) { return w4::run_length(w4::row_tiles(W), a.E, a.topk, a.tn, grid); };
    a.split_up = w4::plan(w4::units(a.up), w4::up_units(FOLD), run(a.up));
    a.split_down = w4::plan(w4::units(a.down), 1, run(a.down));
    const size_t smem = ROOM_BYTES + (size_t(a.tn) * a.topk * 6 + 1 + a.E) * 4;
    constexpr size_t most = ROOM_BYTES + (size_t(T_BLOCK) * K_MAX * 6 + 1 + E_MAX) * 4;
    static std::atomic<int> ready[64];
    once_per_device(ready, [&] { VELA_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(most))); });
    void* args[] = {&a};
    VELA_CUDA(cudaLaunchCooperativeKernel(reinterpret_cast<const void*>(kernel), dim3(grid), dim3(WARPS * 32), args, smem, st));
}
template <class X, int FOLD, bool ZERO> void launch_few(cudaStream_t st, MoeArgs a) {
    auto* up = few_up_kernel<X, FOLD, ZERO>;
    const size_t smem = few::up_bytes<FOLD>(a.T, w4::units(a.up), a.E);
    static std::atomic<int> ready[64];
    once_per_device(ready, [&] { VELA_CUDA(cudaFuncSetAttribute(up, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_SMEM)); });
    // no more clusters than run at a time (71 of 2 x 148 blocks; the others would wait for a whole kernel); all of a block's items
    // in one round if there are warps for it, since a round costs a memory latency
    const int items = a.T * a.topk * w4::row_tiles(a.up);
    const int grid = std::min(ceil_div(items, few::RANKS), clusters_per_device(reinterpret_cast<const void*>(up), few::RANKS, few::WARPS * 32, smem)) * few::RANKS;
    const int ks = std::max(1, std::min(w4::units(a.up), few::WARPS / ceil_div(items, grid)));
    a.split_up = w4::Split{ks, few::WARPS / ks, 1};
    up<<<grid, few::WARPS * 32, smem, st>>>(a);
    // 32 warps on a row tile where there is one for an SM at most, so that each has half as many units one after another (E = 64,
    // D = 2048: 18.6 -> 16.1 us a layer when it was chosen), else two blocks of 16 (D = 4096, where 32 took 22.3 us against 20.8)
    const int rows = a.T * w4::row_tiles(a.down), sms = sm_count();
    const bool wide = rows <= sms && a.topk * w4::units(a.down) > 16;
    // brought up while the first is still running; it waits for it before it reads anything
    cudaLaunchAttribute at[1] = {};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(std::min(rows, 2 * sms)); cfg.blockDim = dim3(wide ? 1024 : 512); cfg.stream = st; cfg.attrs = at; cfg.numAttrs = 1;
    VELA_CUDA(cudaLaunchKernelEx(&cfg, wide ? few_down_kernel<FOLD, ZERO, 32> : few_down_kernel<FOLD, ZERO, 16>, a));
}
template <int FOLD> void launch_few(cudaStream_t st, const MoeArgs& a) {
    if (a.ytype == VELA_T_BF16) a.up.zero ? launch_few<__nv_bfloat16, FOLD, true>(st, a) : launch_few<__nv_bfloat16, FOLD, false>(st, a);
    else a.up.zero ? launch_few<__half, FOLD, true>(st, a) : launch_few<__half, FOLD, false>(st, a);
}
// Which form.  Measured over 1 to 8 tokens, widths 512 to 4096, 8 to 128 experts of 256 to 2048, by the gate and up units of 128
// columns for each SM and one and a half times the units of the tokens' rows, which every block stages: the few-token form takes 7
// to 24 us against 16 to 32 of the other up to 330, and 39 against 38 at 540, 36 against 28 at 490.
template <int FOLD> bool is_few(const MoeArgs& a, int router_type) {
    const double units = double(a.T) * a.topk * w4::row_tiles(a.up) * w4::units(a.up) / sm_count() + 1.5 * a.T * w4::units(a.up);
    return units <= 430 && a.T <= few::TOKENS && a.E <= few::EXPERTS && a.T * a.topk <= few::PAIRS && router_type == a.ytype && a.vecx && a.vecr &&
           size_t(a.E) * a.D <= FEW_ROUTER && few::up_bytes<FOLD>(a.T, w4::units(a.up), a.E) <= FEW_SMEM && !a.extra;
}
template <int FOLD> void launch(cudaStream_t st, MoeArgs a, int router_type) {
    if (is_few<FOLD>(a, router_type)) return launch_few<FOLD>(st, a);
    a.err = device_error_word(&g_moe_err);
    const dim3 grid(RANKS, a.T);
    if (a.ytype == VELA_T_BF16) {
        if (router_type == VELA_T_F32) route_kernel<__nv_bfloat16, float, FOLD><<<grid, ROUTE_WARPS * 32, 0, st>>>(a);
        else route_kernel<__nv_bfloat16, __nv_bfloat16, FOLD><<<grid, ROUTE_WARPS * 32, 0, st>>>(a);
    } else {
        if (router_type == VELA_T_F32) route_kernel<__half, float, FOLD><<<grid, ROUTE_WARPS * 32, 0, st>>>(a);
        else route_kernel<__half, __half, FOLD><<<grid, ROUTE_WARPS * 32, 0, st>>>(a);
    }
    for (a.t0 = 0; a.t0 < a.T; a.t0 += T_BLOCK) {
        a.tn = std::min(T_BLOCK, a.T - a.t0);
        a.up.zero ? launch_experts<FOLD, true>(st, a) : launch_experts<FOLD, false>(st, a);
    }
}

void moe_w4(cudaStream_t st, int type, const void* X, int ldx, int T, const vela_moe& L, void* Y, int ldy, int32_t* ids, float* weights,
            void* ws, size_t bytes, unsigned extra, long long limit) {
    VELA_REQUIRE(type == VELA_T_BF16 || type == VELA_T_F16, "moe_w4: type must be bf16 or f16");
    check(L, T);
    MoeArgs a{};
    a.up = w4_weights(L.gate_up, "moe_w4 gate_up");
    a.down = w4_weights(L.down, "moe_w4 down");
    if (T == 0) return;
    VELA_REQUIRE(X && Y && L.router, "moe_w4: null X, Y or router");
    VELA_REQUIRE(L.router_type == type || L.router_type == VELA_T_F32, "moe_w4: the router must be f32 or of X's type");
    VELA_REQUIRE(ldx >= L.D && ldy >= L.D, "moe_w4: a leading dimension is too small");
    VELA_REQUIRE(aligned(X, 2) && aligned(Y, 2) && aligned(L.router, elem_bytes(L.router_type)) && aligned(L.select_bias, 4) && aligned(ids, 4) &&
                 aligned(weights, 4), "moe_w4: a pointer is not aligned to its type");
    const Layout o = layout(L, T);
    VELA_REQUIRE(ws && aligned(ws, 16) && bytes >= o.bytes, "moe_w4: the workspace is missing, not aligned or too small");
    uint8_t* w = static_cast<uint8_t*>(ws);
    a.X = X; a.router = L.router; a.bias = L.select_bias; a.Y = Y;
    a.ids = ids ? ids : reinterpret_cast<int32_t*>(w + o.ids);
    a.weights = weights ? weights : reinterpret_cast<float*>(w + o.weights);
    a.xs = reinterpret_cast<__half*>(w + o.xs);
    a.xp = reinterpret_cast<float2*>(w + o.xp);
    a.h = reinterpret_cast<float*>(w + o.h);
    a.o = reinterpret_cast<float*>(w + o.o);
    a.hi = reinterpret_cast<__nv_bfloat16*>(w + o.hi);
    a.lo = reinterpret_cast<__nv_bfloat16*>(w + o.lo);
    a.count = reinterpret_cast<unsigned*>(w + o.count);
    a.D = L.D; a.I = L.I; a.E = L.E; a.topk = L.topk; a.T = T; a.ldx = ldx; a.ldy = ldy; a.score = L.score; a.renorm = L.renorm; a.scale = L.scale;
    a.ytype = type;
    a.vecx = L.D % 8 == 0 && ldx % 8 == 0 && aligned(X, 16);
    a.vecr = L.D % 8 == 0 && aligned(L.router, 16);
    a.limit = limit > 0 ? limit : WAIT_LIMIT_CYCLES;
    a.extra = extra;
    if (L.gate_up.group == 32) launch<32>(st, a, L.router_type);
    else if (L.gate_up.group == 64) launch<64>(st, a, L.router_type);
    else launch<128>(st, a, L.router_type);
}
}  // namespace
}  // namespace vela

extern "C" size_t vela_moe_w4_workspace(const vela_moe* L, int T) {
    size_t n = 0;
    vela::guarded_host("vela_moe_w4_workspace", [&] {
        VELA_REQUIRE(L, "moe_w4: null layer");
        vela::check(*L, T);
        n = vela::layout(*L, T > 0 ? T : 1).bytes;
    });
    return n;
}

extern "C" int vela_moe_w4(void* stream, int type, const void* X, int ldx, int T, const vela_moe* L, void* Y, int ldy,
                           int32_t* ids, float* weights, void* workspace, size_t workspace_bytes) {
    return vela::guarded("vela_moe_w4", [&] {
        VELA_REQUIRE(L, "moe_w4: null layer");
        vela::moe_w4(static_cast<cudaStream_t>(stream), type, X, ldx, T, *L, Y, ldy, ids, weights, workspace, workspace_bytes, 0, 0);
    });
}

extern "C" int vela_moe_w4_stalled(void* stream, int type, const void* X, int ldx, int T, const vela_moe* L, void* Y, int ldy,
                                   int32_t* ids, float* weights, void* workspace, size_t workspace_bytes, long long wait_limit_cycles) {
    return vela::guarded("vela_moe_w4_stalled", [&] {
        VELA_REQUIRE(L, "moe_w4: null layer");
        VELA_REQUIRE(wait_limit_cycles > 0, "moe_w4: the wait limit must be positive");
        vela::moe_w4(static_cast<cudaStream_t>(stream), type, X, ldx, T, *L, Y, ldy, ids, weights, workspace, workspace_bytes, 1, wait_limit_cycles);
    });
}
