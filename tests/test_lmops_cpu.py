"""The 4-bit decoding operators without a GPU: the weight layout and its packing, quantisation to the nearest code, struct
layouts, workspace sizes, and arguments that are refused on the host with VELA_ERR_ARG and a message."""
import ctypes

import numpy as np
import pytest

import vela_b200 as V
from vela_b200 import abi


def P(a):
    return None if a is None else a.ctypes.data_as(ctypes.c_void_p)


def bf16(v):
    return (np.asarray(v, np.uint32) << 16).view(np.float32)


def widen(s, scale_type):
    return s.view(np.float16).astype(np.float32) if scale_type == abi.T_F16 else bf16(s.view(np.uint16))


def unpack(q, s, z, N, K, group, scale_type):
    """codes, scales, zeros by the layout's definition, element by element"""
    kt, ng = -(-K // 64), -(-K // group)
    codes = np.zeros((N, K), np.uint8)
    for n in range(N):
        for k in range(K):
            i = k % 64
            h, t, j, b = i // 32, i % 32 // 8, i % 8 // 4, (0, 2, 1, 3).index(i % 4)
            byte = q[((n // 16) * kt + k // 64) * 512 + 16 * (4 * (n % 8) + t) + 8 * h + 4 * j + b]
            codes[n, k] = byte >> 4 if n % 16 >= 8 else byte & 15
    at = np.array([[((n // 16 * ng + g) * 8 + n % 8) * 2 + n // 8 % 2 for g in range(ng)] for n in range(N)])
    return codes, widen(s, scale_type)[at], None if z is None else z[at]


def buffers(N, K, group, zero):
    L = V.lib()
    n = L.vela_w4_scales(N, K, group)
    return np.full(L.vela_w4_bytes(N, K), 0xA5, np.uint8), np.full(n, 0xA5A5, np.uint16), np.full(n, 0xA5, np.uint8) if zero else None


SIZES = [(1, 1, 32), (16, 64, 64), (17, 65, 32), (40, 200, 128), (8, 130, 64), (33, 256, 128)]


@pytest.mark.parametrize("N,K,group", SIZES)
@pytest.mark.parametrize("zero", [False, True])
def test_pack_follows_the_layout(N, K, group, zero):
    r = np.random.default_rng(N + K)
    ng = -(-K // group)
    for scale_type in (abi.T_BF16, abi.T_F16):
        codes = r.integers(0, 16, (N, K)).astype(np.uint8)
        scales = bf16(r.integers(0x3c00, 0x3f00, (N, ng)))       # exact in bf16
        if scale_type == abi.T_F16:
            scales = scales.astype(np.float16).astype(np.float32)
        zeros = r.integers(0, 16, (N, ng)).astype(np.uint8) if zero else None
        q, s, z = buffers(N, K, group, zero)
        V.check(V.lib().vela_w4_pack(P(codes), P(scales), P(zeros), N, K, group, scale_type, P(q), P(s), P(z)))
        c2, s2, z2 = unpack(q, s, z, N, K, group, scale_type)
        assert np.array_equal(c2, codes) and np.array_equal(s2, scales)
        assert z2 is None if zeros is None else np.array_equal(z2, zeros)
        # what is padding is zero: the nibbles and scales that hold no element
        assert int((np.stack([q & 15, q >> 4]) != 0).sum()) == int((codes != 0).sum())
        assert int((s != 0).sum()) == int((scales != 0).sum())


def test_sizes():
    L = V.lib()
    assert L.vela_w4_bytes(16, 64) == 512 and L.vela_w4_bytes(17, 65) == 4 * 512
    assert L.vela_w4_bytes(1 << 20, 1 << 16) == (1 << 35)           # past 32 bits
    assert L.vela_w4_scales(17, 65, 32) == 32 * 3
    for bad in ((0, 64), (16, 0), (-1, 64)):
        assert L.vela_w4_bytes(*bad) == 0 and L.vela_w4_scales(*bad, 64) == 0
    assert L.vela_w4_scales(16, 64, 48) == 0


@pytest.mark.parametrize("N,K,group", SIZES)
@pytest.mark.parametrize("asym", [0, 1])
def test_quantize_takes_the_nearest_code(N, K, group, asym):
    r = np.random.default_rng(N * K)
    W = r.normal(0, 1, (N, K)).astype(np.float32)
    W[0, : min(K, group)] = 0                                       # a group of zeros
    if N > 1:
        W[1] = np.abs(W[1])                                         # a row without negative values
    for scale_type in (abi.T_BF16, abi.T_F16):
        q, s, z = buffers(N, K, group, bool(asym))
        V.check(V.lib().vela_w4_quantize(P(W), N, K, group, asym, scale_type, P(q), P(s), P(z)))
        codes, scales, zeros = unpack(q, s, z, N, K, group, scale_type)
        rep = lambda a: np.repeat(a.astype(np.float64), group, 1)[:, :K]  # noqa: E731
        zz = rep(zeros) if asym else 8.0
        value = (codes.astype(np.float64) - zz) * rep(scales)
        # half a step; the scale's own rounding (2^-9 of it at most) moves the ends of the range by 15 times that, and an
        # asymmetric zero point rounds the range's ends by half a step more
        assert (np.abs(value - W) <= rep(scales) * (0.5 + 15 * 2.0 ** -9 + (0.5 if asym else 0)) + 1e-12).all()
        others = (np.arange(16)[None, None] - (zz[..., None] if asym else 8.0)) * rep(scales)[..., None]
        assert (np.abs(value - W) <= np.abs(others - W[..., None]).min(-1) + 1e-6).all()
        assert (value[0, : min(K, group)] == 0).all()


def test_helpers():
    r = np.random.default_rng(3)
    W = r.normal(0, 1, (24, 96)).astype(np.float32)
    w = V.w4_quantize(W, group=32, asym=True, scale_type="f16")
    codes, scales, zeros = unpack(w["q"], w["scale"], w["zero"], 24, 96, 32, abi.T_F16)
    assert np.abs((codes - np.repeat(zeros, 32, 1).astype(np.float64)) * np.repeat(scales, 32, 1) - W).max() < 0.5
    gate, up = np.arange(16 * 3).reshape(16, 3), 100 + np.arange(16 * 3).reshape(16, 3)
    both = V.moe_gate_up(gate, up)
    assert both.shape == (32, 3)
    assert np.array_equal(both[:8], gate[:8]) and np.array_equal(both[8:16], up[:8]) and np.array_equal(both[24:], up[8:])


def test_struct_layouts():
    assert ctypes.sizeof(abi.W4) == 40 and abi.W4.scale_type.offset == 36
    assert abi.Moe.router.offset == 16 and abi.Moe.select_bias.offset == 32 and abi.Moe.gate_up.offset == 56 and ctypes.sizeof(abi.Moe) == 136


def refused(rc, word):
    msg = V.lib().vela_last_error().decode()
    assert rc == -1, (rc, msg)
    assert word in msg, msg


def test_pack_and_quantize_refuse():
    L = V.lib()
    q, s, z = buffers(16, 64, 64, True)
    codes, sc, ze = np.zeros((16, 64), np.uint8), np.ones((16, 1), np.float32), np.zeros((16, 1), np.uint8)
    args = lambda **k: [{**dict(c=P(codes), s=P(sc), z=None, N=16, K=64, g=64, t=0, q=P(q), so=P(s), zo=None), **k}[n] for n in ("c", "s", "z", "N", "K", "g", "t", "q", "so", "zo")]  # noqa: E731
    assert L.vela_w4_pack(*args()) == 0
    refused(L.vela_w4_pack(*args(c=None)), "null")
    refused(L.vela_w4_pack(*args(N=0)), "N, K > 0")
    refused(L.vela_w4_pack(*args(g=100)), "group")
    refused(L.vela_w4_pack(*args(t=2)), "scales")
    refused(L.vela_w4_pack(*args(z=P(ze))), "zero")
    codes[3, 3] = 16
    refused(L.vela_w4_pack(*args()), "code above 15")
    codes[3, 3] = 0
    ze[1] = 16
    refused(L.vela_w4_pack(*args(z=P(ze), zo=P(z))), "zero point above 15")
    W = np.zeros((16, 64), np.float32)
    assert L.vela_w4_quantize(P(W), 16, 64, 64, 0, 0, P(q), P(s), None) == 0
    refused(L.vela_w4_quantize(P(W), 16, 64, 64, 1, 0, P(q), P(s), None), "zero")
    refused(L.vela_w4_quantize(P(W), 16, 64, 64, 0, 0, P(q), P(s), P(z)), "zero")
    W[2, 2] = np.nan
    refused(L.vela_w4_quantize(P(W), 16, 64, 64, 0, 0, P(q), P(s), None), "not finite")
    W[2, 2] = 1e38
    refused(L.vela_w4_quantize(P(W), 16, 64, 64, 0, 1, P(q), P(s), None), "overflows")


def test_rms_norm_refuses():
    L = V.lib()
    base = dict(type=0, X=64, ldx=64, R=None, ldr=64, g=64, eps=1e-5, M=1, C=64, S=None, lds=64, Y=None, ldy=64, qt=3, Q=64, ldq=64, sc=64, grp=0)
    call = lambda **k: L.vela_rms_norm_q8(None, *{**base, **k}.values())  # noqa: E731
    refused(call(type=3), "type")
    refused(call(C=0), "C > 0")
    refused(call(M=-1), "M >= 0")
    refused(call(X=None), "null")
    refused(call(g=None), "null")
    refused(call(ldx=63), "leading dimension")
    refused(call(R=64, ldr=8), "leading dimension")
    refused(call(ldq=8), "leading dimension")
    refused(call(eps=-1.0), "eps")
    refused(call(eps=float("nan")), "eps")
    refused(call(qt=0), "qtype")
    refused(call(sc=None), "qscale")
    refused(call(grp=32), "qgroup")
    refused(call(X=65), "aligned")
    refused(call(S=64, lds=128), "in place")


def w4(**k):
    d = dict(q=512, scale=512, zero=None, N=64, K=128, group=64, scale_type=0)
    return abi.W4(*{**d, **k}.values())


def test_gemv_refuses():
    L = V.lib()
    base = dict(xt=0, X=64, ldx=128, xs=None, xg=0, M=1, W=w4(), b=None, r=None, ldr=64, yt=0, Y=64, ldy=64)

    def call(**k):
        a = {**base, **k}
        a["W"] = ctypes.byref(a["W"]) if a["W"] is not None else None
        return L.vela_gemv_w4(None, *a.values())
    refused(call(W=None), "null weights")
    refused(call(W=w4(q=None)), "null weights")
    refused(call(W=w4(q=520)), "aligned")
    refused(call(W=w4(group=48)), "group")
    refused(call(W=w4(N=0)), "N, K > 0")
    refused(call(W=w4(scale_type=2)), "bf16 or f16")
    refused(call(xt=2), "X must be")
    refused(call(yt=3), "Y must be")
    refused(call(M=-1), "negative")
    refused(call(X=None), "null X")
    refused(call(Y=None), "null X or Y")
    refused(call(ldx=127), "leading dimension")
    refused(call(ldy=63), "leading dimension")
    refused(call(r=128, ldr=3), "leading dimension")
    refused(call(r=64, ldr=100), "in place")
    refused(call(X=65), "aligned")
    refused(call(xt=3), "xscale")
    refused(call(xt=3, xs=64, xg=32), "xgroup")


def moe(**k):
    d = dict(D=128, I=64, E=4, topk=2, router=64, router_type=0, select_bias=None, score=0, renorm=1, scale=1.0,
             gate_up=w4(N=128, K=128), down=w4(N=128, K=64))
    return abi.Moe(*{**d, **k}.values())


def test_moe_refuses():
    L = V.lib()
    n = L.vela_moe_w4_workspace(ctypes.byref(moe()), 3)
    assert n > 0 and L.vela_moe_w4_workspace(ctypes.byref(moe()), 30) > n
    assert L.vela_moe_w4_workspace(None, 3) == 0 and L.vela_moe_w4_workspace(ctypes.byref(moe()), -1) == 0
    base = dict(type=0, X=64, ldx=128, T=3, L=moe(), Y=64, ldy=128, ids=None, w=None, ws=64, n=n)

    def call(**k):
        a = {**base, **k}
        a["L"] = ctypes.byref(a["L"]) if a["L"] is not None else None
        return L.vela_moe_w4(None, *a.values())
    refused(call(L=None), "null layer")
    refused(call(type=2), "type")
    refused(call(T=-1), "T must")
    refused(call(X=None), "null X")
    refused(call(L=moe(router=None)), "router")
    refused(call(L=moe(router_type=1)), "router")
    refused(call(L=moe(topk=5)), "topk")
    refused(call(L=moe(topk=0)), "topk")
    refused(call(L=moe(E=2000)), "E in")
    refused(call(L=moe(I=60, gate_up=w4(N=120, K=128), down=w4(N=128, K=60))), "multiple of 8")
    refused(call(L=moe(score=2)), "score")
    refused(call(L=moe(gate_up=w4(N=64, K=128))), "gate_up")
    refused(call(L=moe(down=w4(N=128, K=128))), "down")
    refused(call(L=moe(down=w4(N=128, K=64, group=128))), "group")
    refused(call(ldx=100), "leading dimension")
    refused(call(ws=None), "workspace")
    refused(call(ws=72), "workspace")
    refused(call(n=n - 1), "workspace")
    refused(call(Y=65), "aligned")
    for bad in (moe(topk=5), moe(I=0), moe(score=3)):
        assert L.vela_moe_w4_workspace(ctypes.byref(bad), 3) == 0
