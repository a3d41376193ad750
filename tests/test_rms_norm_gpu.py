"""vela_rms_norm_q8 against the formula in 64 bits: every type and 8-bit form, odd widths, strides, in-place residuals,
rows of zeros, NaN and infinities, and widths beyond what a block holds in registers.

Bounds: h is one rounded sum (S: one more rounding to its type).  The mean square is a 32-bit sum of at most 32 values
in a thread and 5 + 16 steps across threads, relative error 64 * 2^-24 at most with the roundings of the square, the mean, the
root and the products; its square root halves it.  y and the scales are held to 64 * 2^-24 relative.  Q stands within half a
step of y / scale: half a unit for int8, 2^-4 of the value (2^-10 where e4m3 is subnormal) for e4m3.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

import vela_b200 as V  # noqa: E402
from vela_b200 import abi  # noqa: E402
from tests.lm_util import DT, ROUND, TINY, ptr, strided, within  # noqa: E402

EPS = 1e-5
REL = 64 * 2.0 ** -24


def call(type, x, r, g, M, C, s, y, qt, q, scale, group, stream=None):
    ld = lambda t: t.stride(0) if t is not None else 0  # noqa: E731
    return V.lib().vela_rms_norm_q8(stream, type, ptr(x), ld(x), ptr(r), ld(r), ptr(g), EPS, M, C, ptr(s), ld(s), ptr(y), ld(y),
                                    qt, ptr(q), ld(q), ptr(scale), group)


def groups(v, group):
    return [v] if not group else list(v.split(group, 1))


def check(type, x, r, g, s, y, qt, q, scale, group, has_s=True):
    h = x.double() + (r.double() if r is not None else 0)
    want = h / torch.sqrt(h.square().mean(1, keepdim=True) + EPS) * g.double()
    if s is not None:
        within(s, h, h.abs() * (ROUND[type] + 2.0 ** -23) + TINY[type], "S")
    if y is not None:
        within(y, want, want.abs() * (ROUND[type] + REL) + TINY[type], "Y")
    if q is not None:
        top = 127.0 if qt == abi.T_I8 else 448.0
        for i, p in enumerate(groups(want, group)):
            a = p.abs().amax(1).clamp_min(1e-30) / top
            within(scale[:, i], a, a * REL, "scale")
            v = q[:, i * group:(i + 1) * group if group else None].to(torch.float32).double()
            t = p / a[:, None]
            if qt == abi.T_I8:
                within(v, t, torch.full_like(t, 0.5 + 127 * 2 * REL), "Q")
                assert v.abs().max() <= 127
            else:
                within(v, t, (t.abs() * (2.0 ** -4 + 2 * REL)).clamp_min(2.0 ** -10 + 1e-6), "Q")


SHAPES = [(1, 1), (1, 7), (3, 8), (1, 64), (5, 130), (2, 333), (77, 1024), (1, 1024), (9, 1031), (4, 2048), (3, 4096), (3, 5000),
          (2, 8192), (2, 12289), (2, 16384), (2, 16392), (1, 20001)]


@pytest.mark.parametrize("type", [abi.T_BF16, abi.T_F16, abi.T_F32])
@pytest.mark.parametrize("M,C", SHAPES)
def test_against_64_bits(type, M, C):
    gen = torch.Generator(device="cuda"); gen.manual_seed(M * 100003 + C)
    for qt in (abi.T_I8, abi.T_E4M3):
        for group in (0, 64, 128):
            for layout in ("plain", "strided", "odd"):
                ld = {"plain": C, "strided": (C + 15) // 8 * 8, "odd": C + 3}[layout]
                off = 1 if layout == "odd" else 0
                ng = -(-C // group) if group else 1
                x, _ = strided(M, C, ld, off, DT[type]); r, _ = strided(M, C, ld, off, DT[type])
                x.copy_(torch.randn(M, C, generator=gen, device="cuda")); r.copy_(3 * torch.randn(M, C, generator=gen, device="cuda"))
                g = (1 + torch.randn(C, generator=gen, device="cuda")).to(DT[type])
                s, sb = strided(M, C, ld, off, DT[type]); y, yb = strided(M, C, ld, off, DT[type]); q, qb = strided(M, C, ld, off, DT[qt])
                scale = torch.empty(M, ng, device="cuda")
                V.check(call(type, x, r, g, M, C, s, y, qt, q, scale, group))
                check(type, x, r, g, s, y, qt, q, scale, group)
                for t, b in ((s, sb), (y, yb), (q, qb)):     # nothing is written between or around the rows
                    b = b.view(torch.uint8).clone().view(-1, t.element_size())
                    idx = torch.arange(b.shape[0], device="cuda") - off
                    inside = (idx >= 0) & (idx < M * ld) & (idx % ld < C)
                    assert (b[~inside] == 0x5A).all()


@pytest.mark.parametrize("type", [abi.T_BF16, abi.T_F32])
@pytest.mark.parametrize("C", [200, 1024, 4096, 20000])
def test_optional_parts_and_in_place(type, C):
    M = 6
    x0 = torch.randn(M, C, device="cuda").to(DT[type]); r0 = torch.randn(M, C, device="cuda").to(DT[type])
    g = torch.randn(C, device="cuda").to(DT[type])
    q = torch.empty(M, C, dtype=torch.int8, device="cuda"); scale = torch.empty(M, 1, device="cuda")
    V.check(call(type, x0, None, g, M, C, None, None, abi.T_I8, q, scale, 0))               # no residual, Q alone
    check(type, x0, None, g, None, None, abi.T_I8, q, scale, 0)
    y = torch.empty_like(x0)
    V.check(call(type, x0, r0, g, M, C, None, y, abi.T_I8, None, None, 0))                  # Y alone
    check(type, x0, r0, g, None, y, abi.T_I8, None, None, 0)
    for which in ("x", "r"):                                                                # the sum over one of its parts
        x, r = x0.clone(), r0.clone()
        s = x if which == "x" else r
        V.check(call(type, x, r, g, M, C, s, None, abi.T_I8, q, scale, 0))
        check(type, x0, r0, g, s, None, abi.T_I8, q, scale, 0)


def test_zero_nan_and_infinite_rows():
    C = 256
    x = torch.randn(5, C, device="cuda"); x[1] = 0; x[2, 7] = float("nan"); x[3, 200] = float("inf"); x[4] *= 1e-38
    g = torch.ones(C, device="cuda")
    for qt in (abi.T_I8, abi.T_E4M3):
        for group in (0, 128):
            ng = 2 if group else 1
            q = torch.empty(5, C, dtype=DT[qt], device="cuda"); scale = torch.empty(5, ng, device="cuda"); y = torch.empty_like(x)
            V.check(call(abi.T_F32, x, None, g, 5, C, None, y, qt, q, scale, group))
            for i in (0, 4):
                check(abi.T_F32, x[i:i + 1], None, g, None, y[i:i + 1], qt, q[i:i + 1], scale[i:i + 1], group)
            assert (y[1] == 0).all() and (q[1].float() == 0).all() and (scale[1] > 0).all()
            assert y[2].isnan().all() and scale[2].isnan().all()
            assert y[3, 200].isnan() and (y[3, :200] == 0).all()
            assert scale[3, -1].isnan() and (group == 0 or scale[3, 0] > 0)


def test_streams_graphs_and_repeats():
    M, C, type = 33, 4096, abi.T_BF16
    x = torch.randn(M, C, device="cuda").bfloat16(); r = torch.randn(M, C, device="cuda").bfloat16(); g = torch.randn(C, device="cuda").bfloat16()
    out = lambda: (torch.empty_like(x), torch.empty(M, C, dtype=torch.int8, device="cuda"), torch.empty(M, 1, device="cuda"))  # noqa: E731
    s, q, scale = out()
    V.check(call(type, x, r, g, M, C, s, None, abi.T_I8, q, scale, 0))
    s2, q2, scale2 = out()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        V.check(call(type, x, r, g, M, C, s2, None, abi.T_I8, q2, scale2, 0, stream=torch.cuda.current_stream().cuda_stream))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(s, s2) and torch.equal(q, q2) and torch.equal(scale, scale2)


def test_no_rows():
    V.check(V.lib().vela_rms_norm_q8(None, abi.T_BF16, None, 64, None, 64, None, EPS, 0, 64, None, 64, None, 64, abi.T_I8, None, 64, None, 0))


@pytest.mark.parametrize("C", [(1 << 31) - 8, (1 << 31) - 1])
def test_the_longest_rows(C):
    """columns up to an int's largest, where a block's stride past the last one is beyond it.  h is +-1 everywhere, so each 32-bit sum of squares is exact
    but for the last ones' rounding, and y = +-2 / sqrt(1 + eps) to the bound of this file; codes are the row's largest, +-127."""
    x = torch.ones(1, C, dtype=torch.bfloat16, device="cuda"); x[0, ::3] = -1
    g = torch.full((C,), 2.0, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(1, C, dtype=torch.bfloat16, device="cuda"); q = torch.zeros(1, C, dtype=torch.int8, device="cuda"); scale = torch.zeros(1, 1, device="cuda")
    V.check(call(abi.T_BF16, x, None, g, 1, C, None, y, abi.T_I8, q, scale, 0))
    a = 2 / (1 + EPS) ** 0.5
    assert abs(scale.item() * 127 / a - 1) <= REL
    for i in range(0, C, 1 << 28):
        sign = x[:, i:i + (1 << 28)].float()
        assert (((y[:, i:i + (1 << 28)].float() * sign - a).abs() <= a * (ROUND[abi.T_BF16] + REL)).all())
        assert (q[:, i:i + (1 << 28)].float() == 127 * sign).all()


def test_the_most_rows():
    """rows up to an int's largest, of the form with several rows a block"""
    M = (1 << 31) - 1
    x = torch.ones(M, 1, dtype=torch.bfloat16, device="cuda"); x[::3] = -1
    g = torch.full((1,), 2.0, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(M, 1, dtype=torch.bfloat16, device="cuda")
    V.check(call(abi.T_BF16, x, None, g, M, 1, None, y, abi.T_I8, None, None, 0))
    a = 2 / (1 + EPS) ** 0.5
    for i in range(0, M, 1 << 28):
        assert (((y[i:i + (1 << 28)].float() * x[i:i + (1 << 28)].float() - a).abs() <= a * (ROUND[abi.T_BF16] + REL)).all())
