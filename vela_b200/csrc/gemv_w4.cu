// Products of a few rows with 4-bit weights: Y[m, n] = sum_k X[m, k] (code - zero) scale + bias + residual.
// A block of 8 warps takes R row tiles (16 R columns of Y) and 8 NT rows of X; its warps share out the tiles along K
// and add their sums in shared memory, in the order of the warps.
#include "host_util.h"
#include "w4.cuh"

namespace vela {
namespace {

constexpr int WARPS = 8;

struct GemvArgs {
    w4::Weights W;
    const void* X; const float* xscale; const float* bias; const void* residual; void* Y;
    int ldx, xgshift, nxg, M, ldr, ldy, ytype;       // xgshift < 0: one scale for each row of X
    bool vec;
};

template <int XT, int NT, int R, bool G32> __global__ void __launch_bounds__(WARPS * 32) gemv_kernel(GemvArgs a) {
    typedef typename w4::Act<XT>::X X;
    constexpr int REGS = w4::Act<XT>::regs;
    __shared__ float red[WARPS][NT * 8][R * 16 + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int rt0 = blockIdx.x * R, m0 = blockIdx.y * NT * 8;
    const int nrt = (a.W.N + 15) / 16;
    const X* xr[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int m = m0 + 8 * n + g;
        xr[n] = m < a.M ? static_cast<const X*>(a.X) + size_t(m) * a.ldx : nullptr;
    }
    float acc[R][NT][4];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.f;

    for (int kt = warp; kt < a.W.kt; kt += WARPS) {
        uint4 w[R];
        w4::ScaleZero sz[R][2];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int rt = min(rt0 + r, nrt - 1);
            w[r] = __ldg(a.W.q + (size_t(rt) * a.W.kt + kt) * 32 + lane);
            sz[r][0] = w4::load_scale(a.W, rt, kt * 64, g);
            if constexpr (G32) sz[r][1] = kt * 64 + 32 < a.W.K ? w4::load_scale(a.W, rt, kt * 64 + 32, g) : sz[r][0];
            else sz[r][1] = sz[r][0];
        }
        uint32_t b[2][NT][REGS];
        float2 sx[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = kt * 64 + 32 * h + 8 * t;
                w4::load_half<XT>(b[h][n], xr[n] ? xr[n] + k : nullptr, a.W.K - k, a.vec);
            }
            sx[n] = make_float2(1.f, 1.f);
            if (w4::Act<XT>::scaled && a.xgshift >= 0) {
                const int m = m0 + 8 * n + 2 * t, i = kt * 64 >> a.xgshift;
                if (m < a.M) sx[n].x = __ldg(a.xscale + size_t(m) * a.nxg + i);
                if (m + 1 < a.M) sx[n].y = __ldg(a.xscale + size_t(m + 1) * a.nxg + i);
            }
        }
        int ones[2][NT][2];
        w4::sums<XT, NT>(ones, b);
#pragma unroll
        for (int r = 0; r < R; ++r) w4::tile<XT, NT, G32>(acc[r], w[r], b, ones, sz[r], sx, a.W.f16);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) red[warp][8 * n + 2 * t + (i & 1)][16 * r + g + 8 * (i >> 1)] = acc[r][n][i];
    __syncthreads();
    for (int i = threadIdx.x; i < NT * 8 * R * 16; i += WARPS * 32) {
        const int c = i % (R * 16), mm = i / (R * 16), n = rt0 * 16 + c, m = m0 + mm;
        if (n >= a.W.N || m >= a.M) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) v += red[w][mm][c];
        if (w4::Act<XT>::scaled && a.xgshift < 0) v *= __ldg(a.xscale + m);
        if (a.bias) v += __ldg(a.bias + n);
        const size_t at = size_t(m) * a.ldy + n, rat = size_t(m) * a.ldr + n;
        if (a.ytype == VELA_T_F32) {
            if (a.residual) v += static_cast<const float*>(a.residual)[rat];
            static_cast<float*>(a.Y)[at] = v;
        } else if (a.ytype == VELA_T_BF16) {
            if (a.residual) v += __bfloat162float(static_cast<const __nv_bfloat16*>(a.residual)[rat]);
            static_cast<__nv_bfloat16*>(a.Y)[at] = __float2bfloat16_rn(v);
        } else {
            if (a.residual) v += __half2float(static_cast<const __half*>(a.residual)[rat]);
            static_cast<__half*>(a.Y)[at] = __float2half_rn(v);
        }
    }
}

template <int XT, int NT, int R> void launch(cudaStream_t st, const GemvArgs& a) {
    const dim3 grid(ceil_div(ceil_div(a.W.N, 16), R), ceil_div(a.M, 8 * NT));
    VELA_REQUIRE(grid.y <= 65535u, "gemv_w4: too many rows");
    if (a.W.gshift == 5) gemv_kernel<XT, NT, R, true><<<grid, WARPS * 32, 0, st>>>(a);
    else gemv_kernel<XT, NT, R, false><<<grid, WARPS * 32, 0, st>>>(a);
}
template <int XT> void launch(cudaStream_t st, const GemvArgs& a) {
    if (a.M <= 8) launch<XT, 1, 1>(st, a);
    else if (a.M <= 16) launch<XT, 2, 1>(st, a);
    else launch<XT, 4, 1>(st, a);
}

void gemv_w4(cudaStream_t st, int xtype, GemvArgs a, int xgroup) {
    const bool scaled = xtype == VELA_T_I8 || xtype == VELA_T_E4M3;
    VELA_REQUIRE(scaled || xtype == VELA_T_BF16 || xtype == VELA_T_F16, "gemv_w4: X must be bf16, f16, int8 or e4m3");
    VELA_REQUIRE(a.ytype == VELA_T_BF16 || a.ytype == VELA_T_F16 || a.ytype == VELA_T_F32, "gemv_w4: Y must be bf16, f16 or f32");
    VELA_REQUIRE(a.M >= 0, "gemv_w4: M must not be negative");
    if (a.M == 0) return;
    VELA_REQUIRE(a.X && a.Y, "gemv_w4: null X or Y");
    VELA_REQUIRE(a.ldx >= a.W.K && a.ldy >= a.W.N && (!a.residual || a.ldr >= a.W.N), "gemv_w4: a leading dimension is too small");
    VELA_REQUIRE(!(a.residual == a.Y && a.ldr != a.ldy), "gemv_w4: the residual in place needs the same ld");
    const size_t xb = elem_bytes(xtype), yb = elem_bytes(a.ytype);
    VELA_REQUIRE(aligned(a.X, xb) && aligned(a.Y, yb) && aligned(a.residual, yb) && aligned(a.bias, 4), "gemv_w4: a pointer is not aligned to its type");
    a.xgshift = -1; a.nxg = 1;
    if (scaled) {
        VELA_REQUIRE(a.xscale && aligned(a.xscale, 4), "gemv_w4: 8-bit X needs xscale");
        VELA_REQUIRE(xgroup == 0 || xgroup == 64 || xgroup == 128, "gemv_w4: xgroup must be 0, 64 or 128");
        if (xgroup) { a.xgshift = xgroup == 64 ? 6 : 7; a.nxg = (a.W.K - 1) / xgroup + 1; }
    }
    a.vec = a.W.K % 8 == 0 && a.ldx % 8 == 0 && aligned(a.X, 8 * xb);
    if (xtype == VELA_T_BF16) launch<VELA_T_BF16>(st, a);
    else if (xtype == VELA_T_F16) launch<VELA_T_F16>(st, a);
    else if (xtype == VELA_T_I8) launch<VELA_T_I8>(st, a);
    else launch<VELA_T_E4M3>(st, a);
}
}  // namespace
}  // namespace vela

extern "C" int vela_gemv_w4(void* stream, int xtype, const void* X, int ldx, const float* xscale, int xgroup, int M, const vela_w4* W,
                            const float* bias, const void* residual, int ldr, int ytype, void* Y, int ldy) {
    return vela::guarded("vela_gemv_w4", [&] {
        VELA_REQUIRE(W, "gemv_w4: null weights");
        vela::GemvArgs a{};
        a.W = vela::w4_weights(*W, "gemv_w4");
        a.X = X; a.xscale = xscale; a.bias = bias; a.residual = residual; a.Y = Y;
        a.ldx = ldx; a.M = M; a.ldr = ldr; a.ldy = ldy; a.ytype = ytype;
        vela::gemv_w4(static_cast<cudaStream_t>(stream), xtype, a, xgroup);
    });
}
