// Residual addition, root-mean-square norm and 8-bit quantisation of rows in one pass:
//   h = X + R,  S = h,  y = h * rsqrt(mean(h^2) + eps) * g,  Y = y,  Q = y / scale.
// h stays in 32-bit registers between the two reductions (the mean square, and the largest |y| of a row or group of columns), so each
// input is read once and each output written once: memory bounds it, from some thousand rows on, and for few rows the launch and one
// memory latency.  8192 x 4096 bf16 with a residual, S and 8-bit groups: 39.5 us, 5.97 TB/s, 93 % of what a copy reaches; 1003 x 5000
// f16 8.9 us (61 %); 77 x 1024 f32 2.3 us.
#include "elem.cuh"
#include "host_util.h"
#include "vela_b200.h"

namespace vela {
namespace {

constexpr float AMAX_MIN = 1e-30f;     // the scale of an all-zero row or group: 127 / AMAX_MIN is still a finite float

struct NormArgs {
    const void* X; const void* R; const void* g; void* S; void* Y; void* Q; float* qscale;
    int ldx, ldr, lds, ldy, ldq, M, C, qgroup, ngroups, gshift, gmask;      // log2 of the group and the group - 1; one group: 31, all bits
    float eps;
};

// over a warp, or over the block through `red` (a word for each warp, not used by the block for anything else)
template <bool WARP, class OP> __device__ __forceinline__ float reduce(float v, float* red, OP op) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (WARP) return v;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int i = 1; i < int(blockDim.x >> 5); ++i) v = op(v, red[i]);
    return v;
}
struct Sum { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };
struct Max { __device__ __forceinline__ float operator()(float a, float b) const { return max_nan(a, b); } };

// 8 values of q = y * inv as bytes
union Bytes8 { uint32_t w[2]; uint8_t b[8]; __nv_fp8x2_storage_t h[4]; };
template <int QT> __device__ __forceinline__ Bytes8 quant8(const float (&y)[8], float inv) {
    Bytes8 o;
    if constexpr (QT == VELA_T_I8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) o.b[i] = uint8_t(max(-127, min(127, __float2int_rn(y[i] * inv))));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) o.h[i] = __nv_cvt_float2_to_fp8x2(make_float2(y[2 * i] * inv, y[2 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    }
    return o;
}
__device__ __forceinline__ void store_q8(uint8_t* p, int n, bool vec, const Bytes8& o) {
    if (vec) *reinterpret_cast<uint2*>(p) = make_uint2(o.w[0], o.w[1]);
    else
#pragma unroll
        for (int i = 0; i < 8; ++i) if (i < n) p[i] = o.b[i];
}

// A block, or with WARP a warp, for each row; thread i holds values 8 (i + j n) .. + 7, j < V, in registers, n the row's threads.
// All three inputs are fetched before the first reduction.  The group of 64 or 128 columns is 8 or 16 neighbouring lanes.  VEC:
// rows are whole and aligned vectors; others are loaded and stored with a warp's 32 elements side by side and brought into the
// lanes' order in shared memory (elem.cuh): 8192 x 4095 bf16 takes 80 us so, 131 with each lane on its own 8 elements (and 126 by
// aligned blocks shifted into place).
//
// MOST: the threads of a block.  Without alignment a block of 1024 is better than four vectors a thread, whose 107 registers leave
// room for one block (2000 x 10241 f16: 79 us against 103); with it the smaller bound is (8192 x 4096 bf16: 39.5 against 40.5).
template <class T, int V, bool WARP, bool VEC> constexpr int MOST = WARP ? 256 : V == 2 && sizeof(T) == 2 && !VEC ? 1024 : 512;
template <class T, int QT, int V, bool WARP, bool VEC> __global__ void __launch_bounds__(MOST<T, V, WARP, VEC>) rms_norm_kernel(const NormArgs a) {
    __shared__ float red[2][MOST<T, V, WARP, VEC> / 32];
    typedef typename Bits<T>::E E;
    __shared__ __align__(16) E lines[VEC ? 1 : MOST<T, V, WARP, VEC> / 32][VEC ? 1 : 256];
    constexpr float TOP = QT == VELA_T_I8 ? 127.f : 448.f;
    const int n = WARP ? 32 : blockDim.x, ti = WARP ? threadIdx.x & 31 : threadIdx.x;
    const size_t row = WARP ? size_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    if (WARP && row >= size_t(a.M)) return;
    const T* x = static_cast<const T*>(a.X) + row * a.ldx;
    const T* r = static_cast<const T*>(a.R) + row * a.ldr;
    const T* g = static_cast<const T*>(a.g);
    Raw8<T> rx[V], rr[V], rg[V];
    const int lane = threadIdx.x & 31;
    E* const line = lines[VEC ? 0 : threadIdx.x >> 5];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = 8 * (ti + j * n), left = a.C - c, c0 = c - 8 * lane;
        if (VEC && left <= 0) { load_raw(rx[j], x, 0, false); load_raw(rr[j], x, 0, false); load_raw(rg[j], g, 0, false); continue; }
        if constexpr (VEC) {
            load_raw(rx[j], x + c, left, true);
            if (a.R) load_raw(rr[j], r + c, left, true);
            load_raw(rg[j], g + c, left, true);
        } else {
            line_load(*reinterpret_cast<Line8<E>*>(&rx[j]), reinterpret_cast<const E*>(x + c0), a.C - c0, lane);
            if (a.R) line_load(*reinterpret_cast<Line8<E>*>(&rr[j]), reinterpret_cast<const E*>(r + c0), a.C - c0, lane);
            line_load(*reinterpret_cast<Line8<E>*>(&rg[j]), reinterpret_cast<const E*>(g + c0), a.C - c0, lane);
        }
    }
    if constexpr (!VEC) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            line_to_lanes(*reinterpret_cast<Line8<E>*>(&rx[j]), line, lane);
            if (a.R) line_to_lanes(*reinterpret_cast<Line8<E>*>(&rr[j]), line, lane);
            line_to_lanes(*reinterpret_cast<Line8<E>*>(&rg[j]), line, lane);
        }
    }
    float h[V][8];
    float ss = 0.f;
    auto store = [&](T* p, int left, const float (&v)[8]) {
        if constexpr (!VEC) {
            Raw8<T> b;
            pack8(b, v);
            line_store(*reinterpret_cast<const Line8<E>*>(&b), reinterpret_cast<E*>(p - 8 * lane), left + 8 * lane, line, lane);
        } else if (left > 0) store8(p, left, true, v);
    };
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = 8 * (ti + j * n);
        unpack8(h[j], rx[j]);
        if (a.R) {
            float t[8];
            unpack8(t, rr[j]);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[j][i] += t[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(h[j][i], h[j][i], ss);
        if (a.S) store(static_cast<T*>(a.S) + row * a.lds + c, a.C - c, h[j]);
    }
    const float rstd = rsqrtf(reduce<WARP>(ss, red[0], Sum()) / float(a.C) + a.eps);
    float top = 0.f, am[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = 8 * (ti + j * n);
        float t[8];
        unpack8(t, rg[j]);
        am[j] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) { h[j][i] = h[j][i] * rstd * t[i]; if (VEC || c + i < a.C) am[j] = max_nan(am[j], fabsf(h[j][i])); }
        if (VEC && c >= a.C) am[j] = 0.f;
        if (a.Y) store(static_cast<T*>(a.Y) + row * a.ldy + c, a.C - c, h[j]);
        top = max_nan(top, am[j]);
    }
    if (!a.Q) return;
    if (a.qgroup == 0) top = reduce<WARP>(top, red[1], Max());
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = 8 * (ti + j * n);
        float m = top;
        if (a.qgroup) {
            m = am[j];
            for (int o = 1; o < 8; o <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (a.gshift == 7) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 8));
        }
        m = m < AMAX_MIN ? AMAX_MIN : m;
        if (c < a.C && (c & a.gmask) == 0) a.qscale[row * a.ngroups + (c >> a.gshift)] = m * (1.f / TOP);
        const Bytes8 q = quant8<QT>(h[j], TOP / m);
        uint8_t* p = static_cast<uint8_t*>(a.Q) + row * a.ldq + c;
        if constexpr (!VEC) {
            Line8<uint8_t> b;
            b.h = make_uint2(q.w[0], q.w[1]);
            line_store(b, p - 8 * lane, a.C - c + 8 * lane, reinterpret_cast<uint8_t*>(line), lane);
        } else if (c < a.C) store_q8(p, a.C - c, true, q);
    }
}

// Rows too long for the registers: the inputs are read again for each step.  S is written last, since it may be X or R.  Columns are
// counted without a sign: a block's stride past the last one may lie beyond 2^31.
template <class T, int QT, int THREADS> __global__ void __launch_bounds__(THREADS) rms_norm_long_kernel(const NormArgs a, bool vec) {
    __shared__ float red[2][THREADS / 32];
    constexpr float TOP = QT == VELA_T_I8 ? 127.f : 448.f;
    const size_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.X) + row * a.ldx;
    const T* r = a.R ? static_cast<const T*>(a.R) + row * a.ldr : nullptr;
    const T* g = static_cast<const T*>(a.g);
    const unsigned C = a.C;
    auto get = [&](unsigned c, int n, float (&h)[8]) {
        load8(x + c, n, vec, h);
        if (r) {
            float t[8];
            load8(r + c, n, vec, t);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] += t[i];
        }
    };
    float ss = 0.f;
    for (unsigned c = 8 * threadIdx.x; c < C; c += 8 * THREADS) {
        float h[8];
        get(c, min(8, int(C - c)), h);
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(h[i], h[i], ss);
    }
    const float rstd = rsqrtf(reduce<false>(ss, red[0], Sum()) / float(a.C) + a.eps);
    float top = 0.f;
    if (a.Q && a.qgroup == 0) {
        for (unsigned c = 8 * threadIdx.x; c < C; c += 8 * THREADS) {
            float h[8], t[8];
            const int n = min(8, int(C - c));
            get(c, n, h);
            load8(g + c, n, vec, t);
#pragma unroll
            for (int i = 0; i < 8; ++i) if (i < n) top = max_nan(top, fabsf(h[i] * rstd * t[i]));
        }
        top = reduce<false>(top, red[1], Max());
    }
    for (unsigned c0 = 0; c0 < C; c0 += 8 * THREADS) {
        const unsigned c = c0 + 8 * threadIdx.x;
        const int n = min(8, int(C - c));                  // negative beyond the row
        float h[8], m = 0.f;
        if (n > 0) {
            float t[8];
            get(c, n, h);
            load8(g + c, n, vec, t);
            if (a.S) store8(static_cast<T*>(a.S) + row * a.lds + c, n, vec, h);
#pragma unroll
            for (int i = 0; i < 8; ++i) { h[i] = h[i] * rstd * t[i]; if (i < n) m = max_nan(m, fabsf(h[i])); }
            if (a.Y) store8(static_cast<T*>(a.Y) + row * a.ldy + c, n, vec, h);
        }
        if (!a.Q) continue;
        if (a.qgroup) { for (int o = 1; o < a.qgroup / 8; o <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o)); }
        else m = top;
        if (n <= 0) continue;
        m = m < AMAX_MIN ? AMAX_MIN : m;
        if ((c & a.gmask) == 0) a.qscale[row * a.ngroups + (c >> a.gshift)] = m * (1.f / TOP);
        store_q8(static_cast<uint8_t*>(a.Q) + row * a.ldq + c, n, vec, quant8<QT>(h, TOP / m));
    }
}

// A warp a row where it has one vector for each lane (8192 x 256 bf16: 3.7 us against 6.1 with a block a row; with two for each
// lane 8192 x 512 takes 7.9 against 8.0, so those go by blocks).  Else a block of as many threads as the row has vectors while
// those are few for the GPU (128 x 4096: 2.6 us against 2.7 with two vectors a thread), and as it has pairs of vectors otherwise
// (256 x 4096: 3.1 against 3.2; 2048 x 4096: 14.2 against 17.0; four a thread: 15.7).  Four where two are not enough for the
// threads (1024 x 16384: 34 us; the kernel for long rows 40).
template <class T, int QT, bool VEC> void launch(cudaStream_t st, const NormArgs& a) {
    const int nv = (a.C - 1) / 8 + 1, warps = 8;
    auto block = [&](int v) { return ceil_div(ceil_div(nv, v), 32) * 32; };
    if (nv <= 32) rms_norm_kernel<T, QT, 1, true, VEC><<<(a.M - 1) / warps + 1, 32 * warps, 0, st>>>(a);
    else if (nv <= 512 && (long long)a.M * nv <= 512 * sm_count()) rms_norm_kernel<T, QT, 1, false, VEC><<<a.M, block(1), 0, st>>>(a);
    else if (nv <= 2 * MOST<T, 2, false, VEC>) rms_norm_kernel<T, QT, 2, false, VEC><<<a.M, block(2), 0, st>>>(a);
    else {
        if constexpr (MOST<T, 2, false, VEC> < 1024) {
            if (nv <= 2048) { rms_norm_kernel<T, QT, 4, false, VEC><<<a.M, block(4), 0, st>>>(a); return; }
        }
        rms_norm_long_kernel<T, QT, 512><<<a.M, 512, 0, st>>>(a, VEC);
    }
}
template <class T, int QT> void launch(cudaStream_t st, const NormArgs& a, bool vec) { vec ? launch<T, QT, true>(st, a) : launch<T, QT, false>(st, a); }

void rms_norm_q8(cudaStream_t st, int type, const NormArgs& a, int qtype) {
    VELA_REQUIRE(type == VELA_T_BF16 || type == VELA_T_F16 || type == VELA_T_F32, "rms_norm_q8: type must be bf16, f16 or f32");
    VELA_REQUIRE(a.M >= 0 && a.C > 0, "rms_norm_q8: M >= 0 and C > 0");
    if (a.M == 0) return;
    VELA_REQUIRE(a.X && a.g, "rms_norm_q8: null X or g");
    VELA_REQUIRE(a.ldx >= a.C && (!a.R || a.ldr >= a.C) && (!a.S || a.lds >= a.C) && (!a.Y || a.ldy >= a.C) && (!a.Q || a.ldq >= a.C),
                 "rms_norm_q8: a leading dimension below C");
    VELA_REQUIRE(a.eps >= 0.f, "rms_norm_q8: eps must not be negative");
    VELA_REQUIRE(!(a.S && ((a.S == a.X && a.lds != a.ldx) || (a.S == a.R && a.lds != a.ldr))), "rms_norm_q8: S in place needs the same ld");
    if (a.Q) {
        VELA_REQUIRE(qtype == VELA_T_I8 || qtype == VELA_T_E4M3, "rms_norm_q8: qtype must be int8 or e4m3");
        VELA_REQUIRE(a.qscale, "rms_norm_q8: Q without qscale");
        VELA_REQUIRE(a.qgroup == 0 || a.qgroup == 64 || a.qgroup == 128, "rms_norm_q8: qgroup must be 0, 64 or 128");
    }
    const size_t b = elem_bytes(type);
    for (const void* p : {a.X, a.R, a.g, static_cast<const void*>(a.S), static_cast<const void*>(a.Y)})
        VELA_REQUIRE(aligned(p, b), "rms_norm_q8: a pointer is not aligned to its type");
    VELA_REQUIRE(aligned(a.qscale, 4), "rms_norm_q8: qscale is not aligned");
    auto row16 = [&](const void* p, int ld) { return !p || (aligned(p, 16) && ld * b % 16 == 0); };
    const bool vec = a.C % 8 == 0 && row16(a.X, a.ldx) && row16(a.R, a.ldr) && row16(a.S, a.lds) && row16(a.Y, a.ldy) && aligned(a.g, 16) &&
                     (!a.Q || (aligned(a.Q, 8) && a.ldq % 8 == 0));
    const bool i8 = qtype == VELA_T_I8;
    if (type == VELA_T_BF16) i8 ? launch<__nv_bfloat16, VELA_T_I8>(st, a, vec) : launch<__nv_bfloat16, VELA_T_E4M3>(st, a, vec);
    else if (type == VELA_T_F16) i8 ? launch<__half, VELA_T_I8>(st, a, vec) : launch<__half, VELA_T_E4M3>(st, a, vec);
    else i8 ? launch<float, VELA_T_I8>(st, a, vec) : launch<float, VELA_T_E4M3>(st, a, vec);
}
}  // namespace
}  // namespace vela

extern "C" int vela_rms_norm_q8(void* stream, int type, const void* X, int ldx, const void* R, int ldr, const void* g, float eps, int M, int C,
                                void* S, int lds, void* Y, int ldy, int qtype, void* Q, int ldq, float* qscale, int qgroup) {
    return vela::guarded("vela_rms_norm_q8", [&] {
        vela::NormArgs a{X, R, g, S, Y, Q, qscale, ldx, ldr, lds, ldy, ldq, M, C, qgroup, qgroup > 0 ? (C - 1) / qgroup + 1 : 1, qgroup == 64 ? 6 : qgroup == 128 ? 7 : 31, qgroup > 0 ? qgroup - 1 : -1, eps};
        vela::rms_norm_q8(static_cast<cudaStream_t>(stream), type, a, qtype);
    });
}
