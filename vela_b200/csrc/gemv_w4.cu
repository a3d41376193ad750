// Products of a few rows with 4-bit weights: Y[m, n] = sum_k X[m, k] (code - zero) scale + bias + residual.
//
// The weights are read once, so with few rows the aim is to keep enough of them in flight and to spend few instructions on each.
// The grid is one wave of 16-warp blocks that stay for the whole call.  Row group (R row tiles) i + j * grid is the j-th of block
// i, so every SM gets about the same number; 2^ksl warps share out a group's units of 128 columns (unit u goes to warp u mod 2^ksl)
// and add their sums in shared memory in the order of the warps.  Each warp loads one unit ahead; the many warps of an SM keep the
// rest in flight (deeper rings in registers or shared memory cost more instructions than the latency that they hide).  Activations
// are read through the L1 cache, which the weights pass by.
//
// What bounds it: the issue of instructions, 140 for a unit of 16 x 128 bf16 codes with their scales (11 of them for each word of 8
// codes), and the latency of the weights.  One row against 32768 x 8192 (139 MB with scales): 32.0 us, 4.3 TB/s, 67 % of what a
// copy reaches (int8 28.9 us); 8192 x 8192 10.3 us, 1024 x 1024 2.5 us, of which a launch and two memory latencies are the most.
// The time hardly grows up to 8 rows (10.6 us).  16 rows take 13.3 us; a profile of it shows the tensor pipe 25 % and issue 32 % busy,
// and of 11 cycles between two instructions of a warp 5 are spent on loads: the 128 registers of two column and two row tiles leave
// room for 16 warps on an SM, too few to hide the latency of the weights and of X, which comes through L1 for every row group.
#include "host_util.h"
#include "w4.cuh"
#include <algorithm>
#include <climits>

namespace vela {
namespace {

constexpr int WARPS = 16;

struct GemvArgs {
    w4::Weights W;
    const void* X; const float* xscale; const float* bias; const void* residual; void* Y;
    int ldx, xgshift, nxg, M, ldr, ldy, ytype;       // xgshift < 0: one scale for each row of X
    int ksl;                                         // log2 of the warps that share a row group
    bool vec;
};

template <int XT> __device__ __forceinline__ void write_y(const GemvArgs& a, int m, int n, float v) {
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

__device__ __forceinline__ void group_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" :: "r"(id), "r"(threads) : "memory"); }

template <int XT, int NT, int R, int BLOCKS, int FOLD, bool ZERO> __global__ void __launch_bounds__(WARPS * 32, BLOCKS) gemv_kernel(const GemvArgs a) {
    typedef typename w4::Act<XT>::X X;
    typedef w4::Unit<FOLD, ZERO> Unit;
    __shared__ float red[WARPS][NT * 8][R * 16 + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int m0 = blockIdx.y * NT * 8;
    const int nrt = w4::row_tiles(a.W), nrg = (nrt + R - 1) / R, nu = w4::units(a.W);
    const int ks = 1 << a.ksl, part = warp & (ks - 1), slots = WARPS >> a.ksl, sl = warp >> a.ksl;
    const w4::Consts k = w4::consts<typename w4::Act<XT>::M>();
    const X* row[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) row[n] = static_cast<const X*>(a.X) + size_t(min(m0 + 8 * n + g, a.M - 1)) * a.ldx + 8 * t;

    const int whole = a.vec ? a.W.K >> 7 : 0;              // units that need no care

    for (int rg = blockIdx.x + gridDim.x * sl; rg < nrg; rg += gridDim.x * slots) {
        float acc[R][NT][4] = {};
        w4::RowPtr at[R];
        const X* x[NT];
        int u = part;
#pragma unroll
        for (int r = 0; r < R; ++r) at[r] = w4::row_ptr(a.W, min(rg * R + r, nrt - 1), u, lane);
#pragma unroll
        for (int n = 0; n < NT; ++n) x[n] = row[n] + size_t(u) * 128;
        auto load = [&](Unit (&s)[R]) {
#pragma unroll
            for (int r = 0; r < R; ++r) { w4::load_unit(s[r], at[r], a.W); w4::advance(at[r], a.W, ks); }
        };
        auto sx = [&](int f, int n) {
            if (a.xgshift < 0) return make_float2(1.f, 1.f);
            const int m = m0 + 8 * n + 2 * t, xi = min((u * 128 + f * FOLD) >> a.xgshift, a.nxg - 1);
            return make_float2(__ldg(a.xscale + size_t(min(m, a.M - 1)) * a.nxg + xi), __ldg(a.xscale + size_t(min(m + 1, a.M - 1)) * a.nxg + xi));
        };
        auto work = [&](const Unit (&s)[R]) {
            w4::unit<XT, true, NT, R>(acc, s, x, 0, a.W.f16, k, sx);
#pragma unroll
            for (int n = 0; n < NT; ++n) x[n] += ks * 128;
            u += ks;
        };
        Unit one[R], two[R];
        if (u < whole) {
            load(one);
            while (true) {
                if (u + ks < whole) load(two);
                work(one);
                if (u >= whole) break;
                if (u + ks < whole) load(one);
                work(two);
                if (u >= whole) break;
            }
        }
        for (; u < nu; u += ks) {
#pragma unroll
            for (int r = 0; r < R; ++r) { w4::load_last(one[r], at[r], a.W, u); w4::advance(at[r], a.W, ks); }
            w4::unit<XT, false, NT, R>(acc, one, x, a.W.K - u * 128 - 8 * t, a.W.f16, k, sx);
#pragma unroll
            for (int n = 0; n < NT; ++n) x[n] += ks * 128;
        }
        if (ks == 1) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int m = m0 + 8 * n + 2 * t + (i & 1), c = (rg * R + r) * 16 + g + 8 * (i >> 1);
                        if (m < a.M && c < a.W.N) write_y<XT>(a, m, c, acc[r][n][i]);
                    }
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) red[warp][8 * n + 2 * t + (i & 1)][16 * r + g + 8 * (i >> 1)] = acc[r][n][i];
            group_sync(sl, ks * 32);
            const int rows = min(NT * 8, a.M - m0);
            for (int i = part * 32 + lane; i < rows * (R * 16); i += ks * 32) {
                const int c = i % (R * 16), mm = i / (R * 16);
                float v = 0.f;
                for (int w = 0; w < ks; ++w) v += red[sl * ks + w][mm][c];
                if (rg * R * 16 + c < a.W.N) write_y<XT>(a, m0 + mm, rg * R * 16 + c, v);
            }
            group_sync(sl, ks * 32);
        }
    }
}

template <int XT, int NT, int R, int BLOCKS, int FOLD, bool ZERO> void launch(cudaStream_t st, GemvArgs a) {
    auto* kernel = gemv_kernel<XT, NT, R, BLOCKS, FOLD, ZERO>;
    const int nrg = ceil_div(w4::row_tiles(a.W), R), nu = w4::units(a.W), mb = ceil_div(a.M, 8 * NT);
    const int wave = std::max(1, sm_count() * blocks_per_sm(reinterpret_cast<const void*>(kernel), WARPS * 32, 0) / mb);
    const dim3 grid(std::min(nrg, wave), mb);
    // the split with the least time: a round costs its longest warp's units and about two more to begin and to meet
    const int per = ceil_div(nrg, int(grid.x));
    a.ksl = 0;
    for (int l = 0, best = INT_MAX; (1 << l) <= WARPS && (1 << l) <= nu; ++l) {
        const int cost = ceil_div(per << l, WARPS) * (ceil_div(nu, 1 << l) + 2);
        if (cost < best) { best = cost; a.ksl = l; }
    }
    kernel<<<grid, WARPS * 32, 0, st>>>(a);
}
template <int XT, int NT, int R, int BLOCKS> void launch(cudaStream_t st, const GemvArgs& a) {
    const int fold = a.W.gshift == 5 ? 32 : a.W.gshift == 6 || a.xgshift == 6 ? 64 : 128;
    if (a.W.zero) {
        if (fold == 32) launch<XT, NT, R, BLOCKS, 32, true>(st, a);
        else if (fold == 64) launch<XT, NT, R, BLOCKS, 64, true>(st, a);
        else launch<XT, NT, R, BLOCKS, 128, true>(st, a);
    } else {
        if (fold == 32) launch<XT, NT, R, BLOCKS, 32, false>(st, a);
        else if (fold == 64) launch<XT, NT, R, BLOCKS, 64, false>(st, a);
        else launch<XT, NT, R, BLOCKS, 128, false>(st, a);
    }
}
// Rows of X at a time, and one or two row tiles to a warp.  Up to 8 rows take one column tile and two blocks on an SM.  Beyond that,
// where there is a second row tile for each SM, two row tiles share what is read of X: 16x8192x8192 bf16 takes 13.2 us with them and
// 16.7 without, 32x8192x8192 (two passes over the weights, the second from L2) 22.6 and 27.5; four column tiles in one pass would
// take 27.5 too.  With few row tiles one is faster (16x2368x4096: 4.3 against 5.1 us).  The rule does not look at K, and loses up to
// 12 % where K is short (16x6000x1024: 4.5 us with two, 4.0 with one; 16x4096x1024 3.60 and 3.36).  17 to 24 rows: three column tiles
// 21.2 us at 24x8192x8192, two passes 22.3.
constexpr int MOST_ROWS = 1 << 19;                         // of one launch: 32768 blocks of 16 along y, which takes 65535
template <int XT> void launch(cudaStream_t st, const GemvArgs& a) {
    if (a.M > MOST_ROWS) {
        const size_t yb = elem_bytes(a.ytype);
        for (int m = 0; m < a.M;) {
            GemvArgs b = a;
            b.M = std::min(MOST_ROWS, a.M - m);
            b.X = static_cast<const typename w4::Act<XT>::X*>(a.X) + size_t(m) * a.ldx;
            if (a.xscale) b.xscale = a.xscale + size_t(m) * a.nxg;
            b.Y = static_cast<uint8_t*>(a.Y) + size_t(m) * a.ldy * yb;
            if (a.residual) b.residual = static_cast<const uint8_t*>(a.residual) + size_t(m) * a.ldr * yb;
            launch<XT>(st, b);
            m += b.M;
        }
        return;
    }
    if (a.M <= 8) launch<XT, 1, 1, 2>(st, a);
    else if (a.M > 16 && a.M <= 24) launch<XT, 3, 1, 1>(st, a);
    else if (w4::row_tiles(a.W) > sm_count()) launch<XT, 2, 2, 1>(st, a);
    else launch<XT, 2, 1, 1>(st, a);
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
    a.vec = a.ldx % 8 == 0 && aligned(a.X, 8 * xb);
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
