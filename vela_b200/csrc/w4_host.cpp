// Host side of the 4-bit weights: sizes, the packing into the tile layout, and quantisation to the nearest code.
#include "w4.cuh"
#include "status.h"
#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>
#include <vector>

namespace vela {
w4::Weights w4_weights(const vela_w4& w, const char* name) {
    const std::string n(name);
    VELA_REQUIRE(w4_sizes_ok(w.N, w.K, w.group), n + ": 4-bit weights need N, K > 0 and a group of 32, 64 or 128");
    VELA_REQUIRE(w.scale_type == VELA_T_BF16 || w.scale_type == VELA_T_F16, n + ": scales must be bf16 or f16");
    VELA_REQUIRE(w.q && w.scale, n + ": null weights or scales");
    VELA_REQUIRE(aligned(w.q, 16) && aligned(w.scale, 16) && aligned(w.zero, 2), n + ": weights or scales are not aligned");
    w4::Weights o;
    o.q = reinterpret_cast<const uint4*>(w.q);
    o.scale = static_cast<const uint32_t*>(w.scale);
    o.zero = reinterpret_cast<const uint16_t*>(w.zero);
    o.N = w.N; o.K = w.K;
    o.kt = (w.K - 1) / 64 + 1;
    o.ng = (w.K - 1) / w.group + 1;
    o.gshift = w.group == 32 ? 5 : w.group == 64 ? 6 : 7;
    o.f16 = w.scale_type == VELA_T_F16;
    return o;
}

namespace {
uint16_t round16(float v, int type) {
    if (type == VELA_T_F16) { const __half h = __float2half_rn(v); uint16_t u; std::memcpy(&u, &h, 2); return u; }
    const __nv_bfloat16 h = __float2bfloat16_rn(v); uint16_t u; std::memcpy(&u, &h, 2); return u;
}
float widen16(uint16_t u, int type) {
    if (type == VELA_T_F16) { __half h; std::memcpy(&h, &u, 2); return __half2float(h); }
    __nv_bfloat16 h; std::memcpy(&h, &u, 2); return __bfloat162float(h);
}
// place of (row, group) among the scales
size_t scale_at(int n, int grp, size_t ng) { return ((size_t(n / 16) * ng + grp) * 8 + n % 8) * 2 + n / 8 % 2; }
// byte of column k in row n; the row's nibble is the high one where n / 8 is odd
size_t code_at(int n, int k, size_t kt) {
    static const int byte_of[4] = {0, 2, 1, 3};
    const int i = k % 64, lane = 4 * (n % 8) + i % 32 / 8;
    return (size_t(n / 16) * kt + k / 64) * 512 + 16 * lane + 8 * (i / 32) + 4 * (i % 8 / 4) + byte_of[i % 4];
}
void check(const char* what, int N, int K, int group, int scale_type) {
    VELA_REQUIRE(w4_sizes_ok(N, K, group), std::string(what) + ": N, K > 0 and a group of 32, 64 or 128");
    VELA_REQUIRE(scale_type == VELA_T_BF16 || scale_type == VELA_T_F16, std::string(what) + ": scales must be bf16 or f16");
}
void put(uint8_t* q, int n, int k, size_t kt, int code) {
    uint8_t& b = q[code_at(n, k, kt)];
    b = uint8_t(n / 8 % 2 ? (b & 0x0f) | code << 4 : (b & 0xf0) | code);
}
}  // namespace
}  // namespace vela

using namespace vela;

extern "C" size_t vela_w4_bytes(int N, int K) { return w4_sizes_ok(N, K, 64) ? w4_bytes(N, K) : 0; }
extern "C" size_t vela_w4_scales(int N, int K, int group) { return w4_sizes_ok(N, K, group) ? w4_scales(N, K, group) : 0; }

extern "C" int vela_w4_pack(const uint8_t* codes, const float* scales, const uint8_t* zeros, int N, int K, int group, int scale_type,
                            uint8_t* q, void* scale, uint8_t* zero) {
    return guarded_host("vela_w4_pack", [&] {
        check("w4_pack", N, K, group, scale_type);
        VELA_REQUIRE(codes && scales && q && scale, "w4_pack: null argument");
        VELA_REQUIRE((zeros != nullptr) == (zero != nullptr), "w4_pack: zero is given exactly where zeros is");
        const size_t ng = (K - 1) / group + 1, kt = (K - 1) / 64 + 1;
        for (size_t i = 0; i < size_t(N) * K; ++i) VELA_REQUIRE(codes[i] <= 15, "w4_pack: a code above 15");
        if (zeros) for (size_t i = 0; i < size_t(N) * ng; ++i) VELA_REQUIRE(zeros[i] <= 15, "w4_pack: a zero point above 15");
        std::memset(q, 0, w4_bytes(N, K));
        std::memset(scale, 0, 2 * w4_scales(N, K, group));
        if (zero) std::memset(zero, 0, w4_scales(N, K, group));
        uint16_t* s = static_cast<uint16_t*>(scale);
        for (int n = 0; n < N; ++n) {
            for (int k = 0; k < K; ++k) put(q, n, k, kt, codes[size_t(n) * K + k]);
            for (size_t g = 0; g < ng; ++g) {
                s[scale_at(n, int(g), ng)] = round16(scales[n * ng + g], scale_type);
                if (zero) zero[scale_at(n, int(g), ng)] = zeros[n * ng + g];
            }
        }
    });
}

extern "C" int vela_w4_quantize(const float* W, int N, int K, int group, int asym, int scale_type, uint8_t* q, void* scale, uint8_t* zero) {
    return guarded_host("vela_w4_quantize", [&] {
        check("w4_quantize", N, K, group, scale_type);
        VELA_REQUIRE(W && q && scale, "w4_quantize: null argument");
        VELA_REQUIRE((asym != 0) == (zero != nullptr), "w4_quantize: zero is given exactly where asym is set");
        const size_t ng = (K - 1) / group + 1, kt = (K - 1) / 64 + 1;
        std::memset(q, 0, w4_bytes(N, K));
        std::memset(scale, 0, 2 * w4_scales(N, K, group));
        if (zero) std::memset(zero, 0, w4_scales(N, K, group));
        uint16_t* s = static_cast<uint16_t*>(scale);
        for (int n = 0; n < N; ++n)
            for (size_t g = 0; g < ng; ++g) {
                const float* w = W + size_t(n) * K;
                const int k0 = int(g) * group, k1 = std::min(K, k0 + group);
                float lo = 0.f, hi = 0.f;
                for (int k = k0; k < k1; ++k) {
                    VELA_REQUIRE(std::isfinite(w[k]), "w4_quantize: a weight is not finite");
                    lo = std::min(lo, w[k]); hi = std::max(hi, w[k]);
                }
                const uint16_t su = round16(asym ? (hi - lo) / 15.f : std::max(-lo, hi) / 7.f, scale_type);
                const float sf = widen16(su, scale_type);
                VELA_REQUIRE(std::isfinite(sf), "w4_quantize: a scale overflows its type");
                int z = 8;
                if (asym) z = sf > 0.f ? std::min(15, std::max(0, int(std::nearbyint(-lo / sf)))) : 0;
                s[scale_at(n, int(g), ng)] = su;
                if (zero) zero[scale_at(n, int(g), ng)] = uint8_t(z);
                for (int k = k0; k < k1; ++k) {
                    const float r = sf > 0.f ? std::nearbyint(w[k] / sf) + float(z) : float(z);
                    put(q, n, k, kt, int(std::min(15.f, std::max(0.f, r))));
                }
            }
    });
}
