// A mixture-of-experts layer for a few tokens on 4-bit weights: routing, the chosen experts' gate and up products with
// silu(gate) * up, and their down products weighed by the router.
#include "host_util.h"
#include "w4.cuh"
#include <climits>

namespace vela {
namespace {

constexpr int WARPS = 8, E_MAX = 1024, K_MAX = 32;

struct MoeArgs {
    w4::Weights up, down;             // expert 0's; the others follow
    const void* X; const void* router; const float* bias; void* Y;
    int32_t* ids; float* weights;     // [T][topk], the caller's or the workspace's
    __nv_bfloat16* hi; __nv_bfloat16* lo;     // [T * topk][I]
    int D, I, E, topk, T, ldx, ldy, score, renorm;
    float scale;
    bool vecx, vecr;
};

template <class X, class RW> __device__ __forceinline__ float dot_row(const X* x, const RW* w, int D, bool vecx, bool vecr, int lane) {
    float s = 0.f;
    for (int k = 8 * lane; k < D; k += 256) {
        float a[8], b[8];
        load8(x + k, min(8, D - k), vecx, a);
        load8(w + k, min(8, D - k), vecr, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(a[i], b[i], s);
    }
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

// One block for each token: the experts' scores, then the choice by one warp.
template <class X, class RW> __global__ void __launch_bounds__(WARPS * 32) route_kernel(MoeArgs a) {
    __shared__ float p[E_MAX], key[E_MAX];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tok = blockIdx.x;
    for (int e = warp; e < a.E; e += WARPS) {
        const float s = dot_row(static_cast<const X*>(a.X) + size_t(tok) * a.ldx, static_cast<const RW*>(a.router) + size_t(e) * a.D, a.D, a.vecx, a.vecr, lane);
        if (lane == 0) p[e] = s;
    }
    __syncthreads();
    if (warp) return;
    if (a.score == 0) {
        float m = -INFINITY;
        for (int e = lane; e < a.E; e += 32) m = fmaxf(m, p[e]);
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        float s = 0.f;
        for (int e = lane; e < a.E; e += 32) s += p[e] = expf(p[e] - m);
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        for (int e = lane; e < a.E; e += 32) p[e] /= s;
    } else {
        for (int e = lane; e < a.E; e += 32) p[e] = 1.f / (1.f + expf(-p[e]));
    }
    for (int e = lane; e < a.E; e += 32) {
        const float v = p[e] + (a.bias ? a.bias[e] : 0.f);
        key[e] = v != v ? -INFINITY : v;
    }
    __syncwarp();
    float mine = 0.f, sum = 0.f;
    int id = 0;
    for (int j = 0; j < a.topk; ++j) {
        float best = -INFINITY;
        int at = INT_MAX;
        for (int e = lane; e < a.E; e += 32) {       // NaN marks an expert that was taken
            const float v = key[e];
            if (v > best || (v == best && e < at)) { best = v; at = e; }
        }
        for (int o = 16; o; o >>= 1) {
            const float v = __shfl_xor_sync(0xffffffffu, best, o);
            const int e = __shfl_xor_sync(0xffffffffu, at, o);
            if (e != INT_MAX && (at == INT_MAX || v > best || (v == best && e < at))) { best = v; at = e; }
        }
        if (lane == 0) key[at] = NAN;
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

// the sums of one row tile of expert e for one activation row, over this warp's tiles; column 0 of the product
template <int XT, bool G32>
__device__ __forceinline__ void one_row(float (&acc)[1][4], const w4::Weights& W, int e, int rt, const typename w4::Act<XT>::X* x, const typename w4::Act<XT>::X* x2,
                                        bool vec, int warp, int lane) {
    const int g = lane >> 2, t = lane & 3, nrt = (W.N + 15) / 16, row = e * nrt + rt;
    for (int kt = warp; kt < W.kt; kt += WARPS) {
        const uint4 w = __ldg(W.q + (size_t(row) * W.kt + kt) * 32 + lane);
        w4::ScaleZero sz[2];
        sz[0] = w4::load_scale(W, row, kt * 64, g);
        sz[1] = G32 && kt * 64 + 32 < W.K ? w4::load_scale(W, row, kt * 64 + 32, g) : sz[0];
        const float2 sx[1] = {make_float2(1.f, 1.f)};
        const int ones[2][1][2] = {};
        for (int part = 0; part < (x2 ? 2 : 1); ++part) {
            const auto* p = part ? x2 : x;
            uint32_t b[2][1][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = kt * 64 + 32 * h + 8 * t;
                w4::load_half<XT>(b[h][0], g == 0 ? p + k : nullptr, W.K - k, vec);
            }
            w4::tile<XT, 1, G32>(acc, w, b, ones, sz, sx, W.f16);
        }
    }
}

template <int XT, bool G32> __global__ void __launch_bounds__(WARPS * 32) up_kernel(MoeArgs a) {
    __shared__ float red[WARPS][16];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int pair = blockIdx.y, tok = pair / a.topk, e = a.ids[pair], rt = blockIdx.x;
    float acc[1][4] = {};
    one_row<XT, G32>(acc, a.up, e, rt, static_cast<const typename w4::Act<XT>::X*>(a.X) + size_t(tok) * a.ldx, nullptr, a.vecx, warp, lane);
    if ((lane & 3) == 0) { red[warp][lane >> 2] = acc[0][0]; red[warp][8 + (lane >> 2)] = acc[0][2]; }
    __syncthreads();
    if (threadIdx.x < 8) {
        float gate = 0.f, up = 0.f;
        for (int w = 0; w < WARPS; ++w) { gate += red[w][threadIdx.x]; up += red[w][8 + threadIdx.x]; }
        const float h = gate / (1.f + expf(-gate)) * up;
        const __nv_bfloat16 hi = __float2bfloat16_rn(h);
        const float hf = __bfloat162float(hi);
        const size_t at = size_t(pair) * a.I + rt * 8 + threadIdx.x;
        a.hi[at] = hi;
        a.lo[at] = __float2bfloat16_rn(isinf(hf) ? 0.f : h - hf);
    }
}

template <class Y, bool G32> __global__ void __launch_bounds__(WARPS * 32) down_kernel(MoeArgs a) {
    __shared__ float red[WARPS][16];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rt = blockIdx.x, tok = blockIdx.y;
    float out[2] = {};
    for (int j = 0; j < a.topk; ++j) {
        const int pair = tok * a.topk + j;
        float acc[1][4] = {};
        one_row<VELA_T_BF16, G32>(acc, a.down, a.ids[pair], rt, a.hi + size_t(pair) * a.I, a.lo + size_t(pair) * a.I, true, warp, lane);
        const float w = a.weights[pair];
        out[0] = fmaf(w, acc[0][0], out[0]);
        out[1] = fmaf(w, acc[0][2], out[1]);
    }
    if ((lane & 3) == 0) { red[warp][lane >> 2] = out[0]; red[warp][8 + (lane >> 2)] = out[1]; }
    __syncthreads();
    const int n = rt * 16 + threadIdx.x;
    if (threadIdx.x < 16 && n < a.D) {
        float v = 0.f;
        for (int w = 0; w < WARPS; ++w) v += red[w][threadIdx.x];
        static_cast<Y*>(a.Y)[size_t(tok) * a.ldy + n] = Elem<Y>::put(v);
    }
}

struct Layout { size_t ids, weights, hi, lo, bytes; };
Layout layout(const vela_moe& L, int T) {
    Layout o;
    const size_t n = size_t(T) * L.topk;
    o.ids = 0;
    o.weights = align_up(n * 4, 256);
    o.hi = o.weights + align_up(n * 4, 256);
    o.lo = o.hi + align_up(n * L.I * 2, 256);
    o.bytes = o.lo + align_up(n * L.I * 2, 256);
    return o;
}

void check(const vela_moe& L, int T) {
    VELA_REQUIRE(T >= 0 && T <= (1 << 20), "moe_w4: T must lie in 0 .. 2^20");
    VELA_REQUIRE(L.D > 0 && L.I > 0 && L.I % 8 == 0 && L.I <= (1 << 24) && L.D <= (1 << 24), "moe_w4: D > 0 and I a positive multiple of 8");
    VELA_REQUIRE(L.E > 0 && L.E <= E_MAX && L.topk > 0 && L.topk <= K_MAX && L.topk <= L.E, "moe_w4: E in 1 .. 1024 and topk in 1 .. min(E, 32)");
    VELA_REQUIRE(L.score == 0 || L.score == 1, "moe_w4: score must be 0 (softmax) or 1 (sigmoid)");
    VELA_REQUIRE(L.gate_up.N == 2 * L.I && L.gate_up.K == L.D, "moe_w4: gate_up must be [2 I, D]");
    VELA_REQUIRE(L.down.N == L.D && L.down.K == L.I, "moe_w4: down must be [D, I]");
    VELA_REQUIRE(L.gate_up.group == L.down.group, "moe_w4: gate_up and down need the same group");
}

template <class T, bool G32> void launch(cudaStream_t st, const MoeArgs& a, int router_type) {
    if (router_type == VELA_T_F32) route_kernel<T, float><<<a.T, WARPS * 32, 0, st>>>(a);
    else route_kernel<T, T><<<a.T, WARPS * 32, 0, st>>>(a);
    up_kernel<Elem<T>::code, G32><<<dim3(a.I / 8, a.T * a.topk), WARPS * 32, 0, st>>>(a);
    down_kernel<T, G32><<<dim3(ceil_div(a.D, 16), a.T), WARPS * 32, 0, st>>>(a);
}

void moe_w4(cudaStream_t st, int type, const void* X, int ldx, int T, const vela_moe& L, void* Y, int ldy, int32_t* ids, float* weights,
            void* ws, size_t bytes) {
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
    a.hi = reinterpret_cast<__nv_bfloat16*>(w + o.hi);
    a.lo = reinterpret_cast<__nv_bfloat16*>(w + o.lo);
    a.D = L.D; a.I = L.I; a.E = L.E; a.topk = L.topk; a.T = T; a.ldx = ldx; a.ldy = ldy; a.score = L.score; a.renorm = L.renorm; a.scale = L.scale;
    a.vecx = L.D % 8 == 0 && ldx % 8 == 0 && aligned(X, 16);
    a.vecr = L.D % 8 == 0 && aligned(L.router, 16);
    const bool g32 = L.gate_up.group == 32;
    if (type == VELA_T_BF16) g32 ? launch<__nv_bfloat16, true>(st, a, L.router_type) : launch<__nv_bfloat16, false>(st, a, L.router_type);
    else g32 ? launch<__half, true>(st, a, L.router_type) : launch<__half, false>(st, a, L.router_type);
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
        vela::moe_w4(static_cast<cudaStream_t>(stream), type, X, ldx, T, *L, Y, ldy, ids, weights, workspace, workspace_bytes);
    });
}
