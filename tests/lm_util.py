"""Helpers of the 4-bit decoding operators' tests: packed weights with their values in 64 bits, and error bounds."""
import ctypes

import numpy as np
import torch

import vela_b200 as V
from vela_b200 import abi

DT = {abi.T_BF16: torch.bfloat16, abi.T_F16: torch.float16, abi.T_F32: torch.float32, abi.T_I8: torch.int8, abi.T_E4M3: torch.float8_e4m3fn}
# half a unit in the last place, relative (7, 10 and 23 stored fraction bits), and the smallest step's half
ROUND = {abi.T_BF16: 2.0 ** -8, abi.T_F16: 2.0 ** -11, abi.T_F32: 2.0 ** -24}
TINY = {abi.T_BF16: 2.0 ** -134, abi.T_F16: 2.0 ** -25, abi.T_F32: 2.0 ** -150}


def ptr(t):
    return None if t is None else t.data_ptr()


def np_ptr(a):
    return None if a is None else a.ctypes.data_as(ctypes.c_void_p)


def pack(codes, scales, zeros, group, scale_type):
    """vela_w4_pack of numpy codes [N, K], scales and zeros [N, groups]: (q, scale, zero) as numpy bytes"""
    L = V.lib()
    N, K = codes.shape
    n = L.vela_w4_scales(N, K, group)
    q, s = np.zeros(L.vela_w4_bytes(N, K), np.uint8), np.zeros(2 * n, np.uint8)
    z = np.zeros(n, np.uint8) if zeros is not None else None
    codes, scales = np.ascontiguousarray(codes, np.uint8), np.ascontiguousarray(scales, np.float32)
    zc = np.ascontiguousarray(zeros, np.uint8) if zeros is not None else None
    V.check(L.vela_w4_pack(np_ptr(codes), np_ptr(scales), np_ptr(zc), N, K, group, scale_type, np_ptr(q), np_ptr(s), np_ptr(z)))
    return q, s, z


class W4:
    """random 4-bit weights: E matrices [N, K] on the GPU and their values in 64 bits, [E, N, K]"""

    def __init__(self, seed, N, K, group, zero, scale_type, E=1, device="cuda"):
        r = np.random.default_rng(seed)
        ng = -(-K // group)
        self.N, self.K, self.group, self.scale_type = N, K, group, scale_type
        qs, ss, zs, vals = [], [], [], []
        for _ in range(E):
            codes = r.integers(0, 16, (N, K)).astype(np.uint8)
            scales = np.exp(r.normal(0, 0.5, (N, ng))).astype(np.float32) / 16
            scales *= np.where(r.random((N, ng)) < 0.1, -1, 1)
            st = torch.from_numpy(scales).to(DT[scale_type])
            zeros = r.integers(0, 16, (N, ng)).astype(np.uint8) if zero else None
            q, s, z = pack(codes, scales, zeros, group, scale_type)
            qs.append(q); ss.append(s); zs.append(z)
            zz = np.repeat(zeros, group, 1)[:, :K].astype(np.float64) if zero else 8.0
            vals.append((codes.astype(np.float64) - zz) * np.repeat(st.double().numpy(), group, 1)[:, :K])
        self.value = torch.from_numpy(np.stack(vals)).to(device)
        self.q, self.s = (torch.from_numpy(np.concatenate(a)).to(device) for a in (qs, ss))
        self.z = torch.from_numpy(np.concatenate(zs)).to(device) if zero else None

    def c(self):
        return abi.W4(ptr(self.q), ptr(self.s), ptr(self.z), self.N, self.K, self.group, self.scale_type)


def strided(M, C, ld, off, dtype, fill=None):
    """an [M, C] view with rows of ld elements that begins `off` elements into its buffer; the buffer is returned too"""
    buf = torch.empty(off + max(M, 1) * ld + 8, dtype=torch.uint8 if dtype in (torch.int8, torch.float8_e4m3fn) else dtype, device="cuda")
    buf.view(torch.uint8).fill_(0x5A)
    buf = buf.view(dtype)
    return buf[off:off + M * ld].view(M, ld)[:, :C], buf


def within(got, want, bound, what=""):
    """|got - want| <= bound everywhere, with a finite `want`"""
    d = (got.double() - want).abs()
    bad = ~(d <= bound)
    assert not bad.any(), "%s: %d of %d values beyond the bound, the worst %.3g times" % (
        what, int(bad.sum()), bad.numel(), float((d / bound.clamp_min(1e-300)).nan_to_num(float("inf")).max()))


def sum_bound(K, mass):
    """error of a 32-bit sum of K products of total magnitude `mass`: a chain of at most 12 additions for each 64 columns
    of a share and one for every tile and share, each at twice a float's rounding (the tensor cores may cut)"""
    return (12 + K / 64 + 16) * 2.0 ** -23 * mass
