// A mixture-of-experts layer for a few tokens on 4-bit weights, in two kernels.
//
// route_kernel: a cluster of 8 blocks for each token scores the experts (a warp for each), chooses, and stages the token's row for the
// products (w4.cuh).  It also clears what the second kernel counts in.
//
// expert_kernel: one wave of blocks (a cooperative launch) does the gate and up products of all chosen experts, meets at a barrier over
// the whole grid, and does the down products.  The tokens of an expert are columns of one product, so its weights are read once for
// every 8 NT of them.  What bounds it is the reading of the chosen experts' weights; the barrier costs about a microsecond, over which
// the first down weights are already under way.
//   Up: an item is one row tile of one expert (8 gate rows and their 8 up rows, so a lane holds both parts of a hidden value); ks
//   warps share its columns.
//   Down: an item is one row tile of the output; its sum runs over all experts' hidden columns, shared out among the block's 16 warps, or
//   those of `split` blocks where there are few row tiles.  Sums are added in a fixed order: the last block to finish a row tile adds the parts.
#include "host_util.h"
#include "tc.cuh"
#include "w4.cuh"
#include <algorithm>
#include <atomic>
#include <climits>
#include <cooperative_groups.h>

namespace vela {
namespace {
namespace cg = cooperative_groups;

constexpr int E_MAX = 1024, K_MAX = 32;
constexpr int T_BLOCK = 32;               // tokens of one expert_kernel launch
constexpr int RANKS = 8, ROUTE_WARPS = 8; // of route_kernel
constexpr int WARPS = 16, BLOCKS = 1;     // of expert_kernel
constexpr int SPLIT_MAX = 4;
static __device__ unsigned g_moe_err;

struct MoeArgs {
    w4::Weights up, down;             // expert 0's; the others follow
    const void* X; const void* router; const float* bias; void* Y;
    int32_t* ids; float* weights;     // [T][topk], the caller's or the workspace's
    __half* xs; float2* xp;           // staged rows [T][units of D], their pairs
    __nv_bfloat16* hi; __nv_bfloat16* lo;     // hidden values [T * topk][units of I]
    float* parts;                     // [SPLIT_MAX][row tiles of D][tokens][16]
    unsigned* count;                  // [launch][1 + row tiles of D]: the grid barrier's, the row tiles'
    int D, I, E, topk, T, ldx, ldy, score, renorm, ytype;
    float scale;
    bool vecx, vecr;
    int t0, tn;                       // expert_kernel: its tokens
    unsigned* err; long long limit; unsigned extra;
};

// sum of 8 products for every lane's 8 columns, W rows of the router at a time
template <class X, class RW> __device__ __forceinline__ float dot_row(const X* x, const RW* w, int D, bool vecx, bool vecr, int lane) {
    float s[4] = {};
    int k = 8 * lane;
    for (; vecx && vecr && k + 3 * 256 < D; k += 4 * 256) {        // D % 8 == 0
        float a[4][8], b[4][8];
#pragma unroll
        for (int j = 0; j < 4; ++j) { load8(w + k + 256 * j, 8, true, b[j]); load8(x + k + 256 * j, 8, true, a[j]); }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) s[j] = fmaf(a[j][i], b[j][i], s[j]);
    }
    for (; k < D; k += 256) {
        float a[8], b[8];
        load8(x + k, min(8, D - k), vecx, a);
        load8(w + k, min(8, D - k), vecr, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) s[0] = fmaf(a[i], b[i], s[0]);
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

template <class X, class RW, int FOLD> __global__ void __cluster_dims__(RANKS, 1, 1) __launch_bounds__(ROUTE_WARPS * 32) route_kernel(const MoeArgs a) {
    __shared__ float p[E_MAX];
    __shared__ uint32_t key[E_MAX];
    cg::cluster_group cluster = cg::this_cluster();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tok = blockIdx.y, rank = blockIdx.x;
    const int gw = rank * ROUTE_WARPS + warp;
    const X* x = static_cast<const X*>(a.X) + size_t(tok) * a.ldx;
    float* lead = cluster.map_shared_rank(p, 0);
    for (int e = gw; e < a.E; e += RANKS * ROUTE_WARPS) {
        const float s = dot_row(x, static_cast<const RW*>(a.router) + size_t(e) * a.D, a.D, a.vecx, a.vecr, lane);
        if (lane == 0) lead[e] = s;
    }
    cluster.sync();
    if (rank != 0 || warp != 0) {
        // all but the choosing warp: the staged row, the hidden rows' padding, the counters
        const int i = gw - 1, n = RANKS * ROUTE_WARPS - 1, nu = w4::units(a.up);
        for (int u = i; u < nu; u += n)
            w4::stage_unit<X, FOLD>(x + u * 128 + 4 * lane, a.D - u * 128 - 4 * lane, a.xs + (size_t(tok) * nu + u) * 128, a.xp + (size_t(tok) * nu + u) * (128 / FOLD), lane);
        const int wide = w4::units(a.down) * 128;
        for (int c = i * 32 + lane; c < a.topk * (wide - a.I); c += n * 32) {
            const size_t at = (size_t(tok) * a.topk + c / (wide - a.I)) * wide + a.I + c % (wide - a.I);
            a.hi[at] = __nv_bfloat16(0.f); a.lo[at] = __nv_bfloat16(0.f);
        }
        if (tok % T_BLOCK == 0) {
            const int per = 1 + w4::row_tiles(a.down);
            for (int c = i * 32 + lane; c < per; c += n * 32) a.count[tok / T_BLOCK * per + c] = 0;
        }
        return;
    }
    if (a.score == 0) {
        float m = -INFINITY, s = 0.f;
        for (int e = lane; e < a.E; e += 32) m = fmaxf(m, p[e]);
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        for (int e = lane; e < a.E; e += 32) s += p[e] = expf(p[e] - m);
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        for (int e = lane; e < a.E; e += 32) p[e] /= s;
    } else {
        for (int e = lane; e < a.E; e += 32) p[e] = 1.f / (1.f + expf(-p[e]));
    }
    for (int e = lane; e < a.E; e += 32) {
        const float v = p[e] + (a.bias ? a.bias[e] : 0.f);
        key[e] = ordered(v != v ? -INFINITY : v);         // above 0, which marks an expert that was taken
    }
    float mine = 0.f, sum = 0.f;
    int id = 0;
    for (int j = 0; j < a.topk; ++j) {
        uint32_t best = 0;
        int at = INT_MAX;
        for (int e = lane; e < a.E; e += 32) if (key[e] > best) { best = key[e]; at = e; }     // the lowest of a lane's largest
        const uint32_t top = __reduce_max_sync(0xffffffffu, best);
        at = __reduce_min_sync(0xffffffffu, best == top ? at : INT_MAX);
        if (at % 32 == lane) key[at] = 0;
        __syncwarp();
        const float w = p[at];
        sum += w;
        if (lane == j) { id = at; mine = w; }
    }
    if (lane < a.topk) {
        a.ids[size_t(tok) * a.topk + lane] = id;
        a.weights[size_t(tok) * a.topk + lane] = (a.renorm ? mine / sum : mine) * a.scale;
    }
}

// The experts that the tokens chose: slot v has expert `expert[v]` and pairs (token * topk + place) list[first[v]] .. list[first[v + 1]), at most `most` of them.
struct Slots {
    int32_t* expert; int32_t* first; int32_t* list; int n;
};

// Shares of `items` items of `nu` units for one of `grid` blocks of WARPS warps: log2 of the warps on an item, so that the rounds take the least
// time.  A round costs its longest warp's units and about two more for meeting.
__device__ __forceinline__ int pick_ksl(int items, int nu, int grid) {
    const int per = (items + grid - 1) / grid;
    int best = 0, cost = INT_MAX;
    for (int l = 0; (1 << l) <= WARPS && (1 << l) <= nu; ++l) {
        const int c = (((per << l) + WARPS - 1) / WARPS) * (((nu + (1 << l) - 1) >> l) + 2);
        if (c < cost) { cost = c; best = l; }
    }
    return best;
}

template <int NT, int FOLD, bool ZERO> __global__ void __launch_bounds__(WARPS * 32, BLOCKS) expert_kernel(const MoeArgs a) {
    typedef w4::Unit<FOLD, ZERO> Unit;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int s_n, s_flag;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int grid = gridDim.x, P = a.tn * a.topk, p0 = a.t0 * a.topk;
    // shared memory: sums [WARPS][max(8 NT, tokens)][17], then the slots
    const int rows = max(8 * NT, a.tn);
    float* red = reinterpret_cast<float*>(smem);
    int32_t* s_list = reinterpret_cast<int32_t*>(red + WARPS * rows * 17);
    int32_t* s_ids = s_list + P;
    int32_t* s_expert = s_ids + P;
    int32_t* s_first = s_expert + P;
    int32_t* s_cnt = s_first + P + 1;
    float* s_w = reinterpret_cast<float*>(s_cnt + a.E);

    for (int e = threadIdx.x; e < a.E; e += WARPS * 32) s_cnt[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < P; i += WARPS * 32) {
        const int e = a.ids[p0 + i];
        s_ids[i] = e;
        s_w[i] = a.weights[p0 + i];
        atomicAdd(s_cnt + e, 1);
    }
    __syncthreads();
    if (warp == 0) {                                // first places and slots, by expert; s_cnt becomes the first place
        int n = 0, at = 0;
        for (int e0 = 0; e0 < a.E; e0 += 32) {
            const int e = e0 + lane, c = e < a.E ? s_cnt[e] : 0, v = (c + 8 * NT - 1) / (8 * NT);
            int ci = c, vi = v;
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, ci, o), y = __shfl_up_sync(0xffffffffu, vi, o);
                if (lane >= o) { ci += x; vi += y; }
            }
            for (int i = 0; i < v; ++i) { s_expert[n + vi - v + i] = e; s_first[n + vi - v + i] = at + ci - c + i * 8 * NT; }
            if (e < a.E) s_cnt[e] = at + ci - c;
            n += __shfl_sync(0xffffffffu, vi, 31);
            at += __shfl_sync(0xffffffffu, ci, 31);
        }
        if (lane == 0) { s_n = n; s_first[n] = at; }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < P; i += WARPS * 32) {
        const int e = s_ids[i];
        int r = 0;
        for (int q = 0; q < i; ++q) r += s_ids[q] == e;
        s_list[s_cnt[e] + r] = i;
    }
    __syncthreads();
    const int V = s_n;

    // ------------------------------------------------ gate and up
    {
        const int rt_up = w4::row_tiles(a.up), nu = w4::units(a.up), items = V * rt_up, whole = a.D >> 7;
        const int ksl = pick_ksl(items, nu, grid), ks = 1 << ksl, part = warp & (ks - 1), sl = warp >> ksl, slots = WARPS >> ksl;
        const int wide = w4::units(a.down) * 128;
        int it = blockIdx.x + grid * sl;
        w4::RowPtr at;
        auto seek = [&](int i) { const int v = i / rt_up; at = w4::row_ptr(a.up, size_t(s_expert[v]) * rt_up + (i - v * rt_up), part, lane); };
        auto fetch = [&](Unit& s, int u) {
            if (u < whole) w4::load_unit(s, at, a.up);
            else w4::load_last(s, at, a.up, u);
            w4::advance(at, a.up, ks);
        };
        Unit one, two;
        if (it < items) { seek(it); fetch(one, part); }
        for (int base = blockIdx.x; base < items; base += grid * slots, it += grid * slots) {
            float acc[NT][4] = {};
            int v = 0, c = 0;
            if (it < items) {
                v = it / rt_up;
                c = s_first[v + 1] - s_first[v];
                const int nt = (c + 7) >> 3;
                const __half* x[NT];
                const float2* pair[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    auto tok = [&](int col) { return size_t(a.t0 + s_list[s_first[v] + min(col, c - 1)] / a.topk); };
                    x[n] = a.xs + (tok(8 * n + g) * nu + part) * 128 + 8 * t;
                    pair[n][0] = a.xp + (tok(8 * n + 2 * t) * nu + part) * (128 / FOLD);
                    pair[n][1] = a.xp + (tok(8 * n + 2 * t + 1) * nu + part) * (128 / FOLD);
                }
                int u = part;
                auto step = [&](const Unit& cur, Unit& nxt) {
                    if (u + ks < nu) fetch(nxt, u + ks);
                    w4::unit_staged<NT, FOLD, ZERO>(acc, cur, x, pair, nt, a.up.f16);
                    u += ks;
#pragma unroll
                    for (int n = 0; n < NT; ++n) { x[n] += ks * 128; pair[n][0] += ks * (128 / FOLD); pair[n][1] += ks * (128 / FOLD); }
                };
                while (true) {
                    step(one, two);
                    if (u >= nu) break;
                    step(two, one);
                    if (u >= nu) break;
                }
                if (it + grid * slots < items) { seek(it + grid * slots); fetch(one, part); }
            }
            auto put = [&](int col, int i, float gate, float up) {       // hidden value i of column col
                const float h = gate / (1.f + expf(-gate)) * up;
                const __nv_bfloat16 hi = __float2bfloat16_rn(h);
                const float hf = __bfloat162float(hi);
                const size_t at = size_t(p0 + s_list[s_first[v] + col]) * wide + (it - v * rt_up) * 8 + i;
                a.hi[at] = hi;
                a.lo[at] = __float2bfloat16_rn(isinf(hf) ? 0.f : h - hf);
            };
            if (ks == 1) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) { const int col = 8 * n + 2 * t + i; if (col < c) put(col, g, acc[n][i], acc[n][i + 2]); }
            } else {
                if (it < items)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) red[(warp * rows + 8 * n + 2 * t + (i & 1)) * 17 + g + 8 * (i >> 1)] = acc[n][i];
                __syncthreads();
                if (it < items)
                    for (int q = part * 32 + lane; q < c * 8; q += ks * 32) {
                        float gate = 0.f, up = 0.f;
                        for (int w = 0; w < ks; ++w) {
                            const float* r = red + ((sl * ks + w) * rows + (q >> 3)) * 17;
                            gate += r[q & 7]; up += r[8 + (q & 7)];
                        }
                        put(q >> 3, q & 7, gate, up);
                    }
                __syncthreads();
            }
        }
    }

    // ------------------------------------------------ down: what is fetched first does not depend on the hidden values
    const int rt_down = w4::row_tiles(a.down), nu = w4::units(a.down), total = V * nu, whole = a.I >> 7;
    int split = 1;
    while (split < SPLIT_MAX && rt_down * split * 2 <= grid && total >= split * 2 * WARPS) split *= 2;
    const int items = rt_down * split;
    const w4::Consts k = w4::consts<__nv_bfloat16>();
    Unit one, two;
    w4::RowPtr at;
    auto span = [&](int s, int w) { return int((long long)total * (s * WARPS + w) / (split * WARPS)); };
    auto fetch = [&](Unit& s, int rt, int q, bool seek) {
        const int v = q / nu, u = q - v * nu;
        if (seek || u == 0) at = w4::row_ptr(a.down, size_t(s_expert[v]) * rt_down + rt, u, lane);
        if (u < whole) w4::load_unit(s, at, a.down);
        else w4::load_last(s, at, a.down, u);
        w4::advance(at, a.down, 1);
    };
    {
        const int s = blockIdx.x / rt_down, q = span(s, warp);
        if (int(blockIdx.x) < items && q < span(s, warp + 1)) fetch(one, blockIdx.x - s * rt_down, q, true);
    }

    // ------------------------------------------------ all hidden values are written
    unsigned* count = a.count + a.t0 / T_BLOCK * (1 + rt_down);
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        atomicAdd(count, 1u);
        s_flag = 0;
        const long long t0 = clock64();
        volatile unsigned* c = count;
        while (*c < grid + a.extra)
            if (clock64() - t0 > a.limit) { atomicCAS(a.err, 0u, unsigned(DEVERR_TIMEOUT_OTHER)); s_flag = 1; break; }
        __threadfence();
    }
    __syncthreads();
    if (s_flag) return;

    for (int it = blockIdx.x; it < items; it += grid) {
        const int s = it / rt_down, rt = it - s * rt_down, end = span(s, warp + 1);
        int q = span(s, warp);
        float* mine = red + warp * rows * 17;          // [token][17]
        for (int i = lane; i < a.tn * 17; i += 32) mine[i] = 0.f;
        __syncwarp();
        if (it != int(blockIdx.x) && q < end) fetch(one, rt, q, true);
        float acc[NT][4] = {};
        const __nv_bfloat16* hi[NT];
        const __nv_bfloat16* lo[NT];
        bool fresh = true;
        auto step = [&](const Unit& cur, Unit& nxt) {
            if (q + 1 < end) fetch(nxt, rt, q + 1, false);
            const int v = q / nu, u = q - v * nu, c = s_first[v + 1] - s_first[v], nt = (c + 7) >> 3;
            if (fresh) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const size_t r = (size_t(p0 + s_list[s_first[v] + min(8 * n + g, c - 1)]) * nu + u) * 128 + 8 * t;
                    hi[n] = a.hi + r; lo[n] = a.lo + r;
                }
                fresh = false;
            }
            w4::unit_two<NT, FOLD, ZERO>(acc, cur, hi, lo, nt, a.down.f16, k);
#pragma unroll
            for (int n = 0; n < NT; ++n) { hi[n] += 128; lo[n] += 128; }
            ++q;
            if (u + 1 < nu && q < end) return;
            fresh = true;                              // the expert's last unit here: its tokens' sums, weighed
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int col = 8 * n + 2 * t + (i & 1);
                    if (col < c) {
                        const int p = s_list[s_first[v] + col];
                        float* d = mine + (p / a.topk) * 17 + g + 8 * (i >> 1);
                        *d = fmaf(s_w[p], acc[n][i], *d);
                    }
                    acc[n][i] = 0.f;
                }
            __syncwarp();
        };
        while (q < end) {
            step(one, two);
            if (q >= end) break;
            step(two, one);
        }
        __syncthreads();
        auto write = [&](int i, float v) {
            const int n = rt * 16 + (i & 15);
            if (n >= a.D) return;
            const size_t at = size_t(a.t0 + (i >> 4)) * a.ldy + n;
            if (a.ytype == VELA_T_BF16) static_cast<__nv_bfloat16*>(a.Y)[at] = __float2bfloat16_rn(v);
            else static_cast<__half*>(a.Y)[at] = __float2half_rn(v);
        };
        const size_t part = size_t(rt_down) * a.tn * 16;
        for (int i = threadIdx.x; i < a.tn * 16; i += WARPS * 32) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) v += red[(w * rows + (i >> 4)) * 17 + (i & 15)];
            if (split == 1) write(i, v);
            else a.parts[s * part + size_t(rt) * a.tn * 16 + i] = v;
        }
        if (split > 1) {
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) s_flag = atomicAdd(count + 1 + rt, 1u) == unsigned(split - 1);
            __syncthreads();
            if (s_flag) {                              // the last of the row tile's blocks
                __threadfence();
                for (int i = threadIdx.x; i < a.tn * 16; i += WARPS * 32) {
                    float v = 0.f;
                    for (int z = 0; z < split; ++z) v += __ldcg(a.parts + z * part + size_t(rt) * a.tn * 16 + i);
                    write(i, v);
                }
            }
        }
        __syncthreads();
    }
}

struct Layout { size_t ids, weights, xs, xp, hi, lo, parts, count, bytes; };
Layout layout(const vela_moe& L, int T) {
    Layout o;
    const size_t n = size_t(T) * L.topk, nu = (size_t(L.D) + 127) / 128, nh = (size_t(L.I) + 127) / 128, rt = (size_t(L.D) + 15) / 16, fold = 128 / L.gate_up.group;
    size_t at = 0;
    auto take = [&](size_t b) { const size_t r = at; at += align_up(b, 256); return r; };
    o.ids = take(n * 4); o.weights = take(n * 4);
    o.xs = take(T * nu * 256); o.xp = take(T * nu * fold * 8);
    o.hi = take(n * nh * 256); o.lo = take(n * nh * 256);
    o.parts = take(SPLIT_MAX * rt * std::min(T, T_BLOCK) * 64);
    o.count = take((size_t(T) + T_BLOCK - 1) / T_BLOCK * (1 + rt) * 4);
    o.bytes = at;
    return o;
}

void check(const vela_moe& L, int T) {
    VELA_REQUIRE(T >= 0 && T <= 65535, "moe_w4: T must lie in 0 .. 65535");
    VELA_REQUIRE(L.D > 0 && L.I > 0 && L.I % 8 == 0 && L.I <= (1 << 24) && L.D <= (1 << 24), "moe_w4: D > 0 and I a positive multiple of 8");
    VELA_REQUIRE(L.E > 0 && L.E <= E_MAX && L.topk > 0 && L.topk <= K_MAX && L.topk <= L.E, "moe_w4: E in 1 .. 1024 and topk in 1 .. min(E, 32)");
    VELA_REQUIRE(L.score == 0 || L.score == 1, "moe_w4: score must be 0 (softmax) or 1 (sigmoid)");
    VELA_REQUIRE(L.gate_up.N == 2 * L.I && L.gate_up.K == L.D, "moe_w4: gate_up must be [2 I, D]");
    VELA_REQUIRE(L.down.N == L.D && L.down.K == L.I, "moe_w4: down must be [D, I]");
    VELA_REQUIRE(L.gate_up.group == L.down.group && w4_sizes_ok(16, 16, L.down.group), "moe_w4: gate_up and down need the same group of 32, 64 or 128");
    VELA_REQUIRE((L.gate_up.zero != nullptr) == (L.down.zero != nullptr), "moe_w4: gate_up and down both have zero points or neither");
}

template <int NT, int FOLD, bool ZERO> void launch_experts(cudaStream_t st, MoeArgs a) {
    auto* kernel = expert_kernel<NT, FOLD, ZERO>;
    const int rows = std::max(8 * NT, a.tn), P = a.tn * a.topk;
    const size_t smem = size_t(WARPS) * rows * 17 * 4 + (size_t(P) * 5 + 1 + a.E) * 4;
    constexpr size_t most = size_t(WARPS) * T_BLOCK * 17 * 4 + (size_t(T_BLOCK) * K_MAX * 5 + 1 + E_MAX) * 4;
    static std::atomic<int> ready[64];
    once_per_device(ready, [&] { VELA_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(most))); });
    const int wave = sm_count() * blocks_per_sm(reinterpret_cast<const void*>(kernel), WARPS * 32, smem);
    void* args[] = {&a};
    VELA_CUDA(cudaLaunchCooperativeKernel(reinterpret_cast<const void*>(kernel), dim3(wave), dim3(WARPS * 32), args, smem, st));
}
template <int FOLD> void launch(cudaStream_t st, MoeArgs a, int router_type) {
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
        if (a.up.zero) a.tn <= 8 ? launch_experts<1, FOLD, true>(st, a) : launch_experts<2, FOLD, true>(st, a);
        else a.tn <= 8 ? launch_experts<1, FOLD, false>(st, a) : launch_experts<2, FOLD, false>(st, a);
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
    a.hi = reinterpret_cast<__nv_bfloat16*>(w + o.hi);
    a.lo = reinterpret_cast<__nv_bfloat16*>(w + o.lo);
    a.parts = reinterpret_cast<float*>(w + o.parts);
    a.count = reinterpret_cast<unsigned*>(w + o.count);
    a.D = L.D; a.I = L.I; a.E = L.E; a.topk = L.topk; a.T = T; a.ldx = ldx; a.ldy = ldy; a.score = L.score; a.renorm = L.renorm; a.scale = L.scale;
    a.ytype = type;
    a.vecx = L.D % 8 == 0 && ldx % 8 == 0 && aligned(X, 16);
    a.vecr = L.D % 8 == 0 && aligned(L.router, 16);
    a.err = device_error_word(&g_moe_err);
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
