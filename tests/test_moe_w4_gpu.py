"""vela_moe_w4 against the layer in 64 bits: routing by softmax and sigmoid, ties, selection bias, one token to many, odd
sizes, group sizes, types, strides, NaN scores, and the whole layer's output.

Bounds, carried through the formula: a score is a 32-bit sum (tests/lm_util.sum_bound), its probability off by that much
relatively (and the normalising sum by as much again); a gate and an up value are 32-bit sums; |d silu| <= 1.1; the hidden
value is kept to 2^-16; the down product is a 32-bit sum once more; Y's type rounds once.
"""
import ctypes

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

import vela_b200 as V  # noqa: E402
from vela_b200 import abi  # noqa: E402
from tests.lm_util import DT, ROUND, TINY, W4, ptr, strided, sum_bound, within  # noqa: E402


class Layer:
    def __init__(self, seed, D, I, E, k, type, group, zero=False, score=0, renorm=1, scale=1.0, bias=False, router_f32=False):
        gen = torch.Generator(device="cuda"); gen.manual_seed(seed)
        self.D, self.I, self.E, self.k, self.type, self.score, self.renorm, self.scale = D, I, E, k, type, score, renorm, scale
        self.router = (torch.randn(E, D, generator=gen, device="cuda") * 2 / D ** 0.5).to(torch.float32 if router_f32 else DT[type])
        self.bias = torch.randn(E, generator=gen, device="cuda") * 0.2 if bias else None
        st = abi.T_F16 if seed % 2 else abi.T_BF16
        self.up, self.down = W4(seed, 2 * I, D, group, zero, st, E), W4(seed + 1, D, I, group, zero, st, E)

    def c(self):
        return abi.Moe(self.D, self.I, self.E, self.k, ptr(self.router), abi.T_F32 if self.router.dtype == torch.float32 else self.type, ptr(self.bias),
                       self.score, self.renorm, self.scale, self.up.c(), self.down.c())

    def __call__(self, x, y, ids=None, w=None, stream=None, ws=None, T=None, ldx=None, ldy=None):
        c = self.c()
        T = x.shape[0] if T is None else T
        n = V.lib().vela_moe_w4_workspace(ctypes.byref(c), T)
        assert n > 0
        if ws is None:
            ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")       # its contents need no preparation
        V.check(V.lib().vela_moe_w4(stream, self.type, ptr(x), ldx or x.stride(0), T, ctypes.byref(c), ptr(y), ldy or y.stride(0), ptr(ids), ptr(w), ptr(ws), n))
        return ws

    def route(self, x):
        """probabilities in 64 bits, their relative error bound, and what the choice goes by"""
        r = self.router.double()
        z = x @ r.t()
        dz = sum_bound(self.D, x.abs() @ r.abs().t())
        p = torch.softmax(z, 1) if self.score == 0 else torch.sigmoid(z)
        rel = 2 * dz.amax(1, keepdim=True) + 2.0 ** -20
        return p, rel, p if self.bias is None else p + self.bias.double()

    def check(self, x, y, ids, w):
        x = x.double()
        T = x.shape[0]
        p, rel, pick = self.route(x)
        want_ids = torch.sort(pick, dim=1, descending=True, stable=True).indices[:, :self.k]
        if ids is not None:     # the inputs keep the choices further apart than the bound
            assert torch.equal(ids.long(), want_ids)
        ww = p.gather(1, want_ids)
        if self.renorm:
            ww = ww / ww.sum(1, keepdim=True)
        ww = ww * self.scale
        if w is not None:
            within(w, ww, ww.abs() * (2 * rel) + 1e-30, "weights")
        want = torch.zeros(T, self.D, dtype=torch.float64, device="cuda")
        bound = torch.zeros_like(want)
        i = torch.arange(self.I, device="cuda")
        gi = i // 8 * 16 + i % 8
        for t in range(T):
            for j in range(self.k):
                e = int(want_ids[t, j])
                u, d = self.up.value[e], self.down.value[e]
                v, mass = u @ x[t], u.abs() @ x[t].abs()
                gate, up, dg, du = v[gi], v[gi + 8], sum_bound(self.D, mass[gi]), sum_bound(self.D, mass[gi + 8])
                s = gate * torch.sigmoid(gate)
                h = s * up
                dh = 1.1 * dg * (up.abs() + du) + s.abs() * du + h.abs() * 2.0 ** -16 + TINY[abi.T_BF16]
                o, om = d @ h, d.abs() @ h.abs()
                do = d.abs() @ dh + sum_bound(self.I * self.k, om)
                want[t] += ww[t, j] * o
                bound[t] += ww[t, j].abs() * (do + 2 * rel[t] * o.abs())
        within(y, want, bound + want.abs() * ROUND[self.type] + TINY[self.type], "Y")


CASES = [
    # T, D, I, E, k, type, group, zero, score, renorm, bias, router_f32
    (1, 64, 32, 4, 1, abi.T_BF16, 32, False, 0, 1, False, False),
    (1, 1024, 512, 16, 2, abi.T_BF16, 128, False, 0, 1, False, False),
    (2, 72, 8, 3, 3, abi.T_F16, 64, True, 1, 0, True, False),
    (3, 333, 40, 7, 2, abi.T_BF16, 32, True, 0, 0, False, True),
    (5, 1288, 648, 10, 3, abi.T_F16, 64, True, 1, 0, True, False),
    (8, 256, 128, 64, 8, abi.T_BF16, 128, False, 0, 1, False, True),
    (9, 200, 264, 5, 4, abi.T_F16, 128, True, 1, 1, False, False),
    (16, 320, 96, 2, 2, abi.T_BF16, 64, False, 0, 1, False, False),
    (17, 130, 24, 33, 5, abi.T_BF16, 32, False, 1, 1, True, True),
    (32, 512, 256, 8, 4, abi.T_BF16, 128, False, 0, 1, False, False),
    (33, 96, 16, 1, 1, abi.T_F16, 64, False, 0, 1, False, False),
    (70, 128, 64, 12, 6, abi.T_BF16, 64, True, 0, 0, False, False),
    (4, 64, 64, 300, 32, abi.T_BF16, 64, False, 0, 1, False, False),
]


@pytest.mark.parametrize("T,D,I,E,k,type,group,zero,score,renorm,bias,f32", CASES)
def test_against_64_bits(T, D, I, E, k, type, group, zero, score, renorm, bias, f32):
    layer = Layer(T + D + I + E, D, I, E, k, type, group, zero, score, renorm, 1.5 if score else 1.0, bias, f32)
    for layout in ("plain", "odd"):
        ld, off = (D, 0) if layout == "plain" else (D + 3, 1)
        gen = torch.Generator(device="cuda"); gen.manual_seed(D + off)
        x, _ = strided(T, D, ld, off, DT[type]); y, yb = strided(T, D, ld, off, DT[type])
        x.copy_(torch.randn(T, D, generator=gen, device="cuda"))
        ids = torch.full((T, k), -1, dtype=torch.int32, device="cuda"); w = torch.full((T, k), float("nan"), device="cuda")
        layer(x, y, ids, w, ldx=ld, ldy=ld)
        layer.check(x, y, ids, w)
        idx = torch.arange(yb.numel(), device="cuda") - off
        inside = (idx >= 0) & (idx < T * ld) & (idx % ld < D)
        assert (yb.view(torch.uint8).view(yb.numel(), -1)[~inside] == 0x5A).all(), "written outside Y"
        y2 = torch.empty(T, D, dtype=DT[type], device="cuda")
        layer(x, y2, ldx=ld)              # without ids and weights, in a fresh workspace: the same bits
        assert torch.equal(y2, y)


def test_ties_go_to_the_lower_expert():
    layer = Layer(5, 64, 16, 12, 5, abi.T_BF16, 64)
    layer.router[:] = layer.router[0].clone()
    layer.router[7] = 0
    x = torch.randn(3, 64, device="cuda").bfloat16()
    y = torch.empty_like(x); ids = torch.empty(3, 5, dtype=torch.int32, device="cuda")
    layer(x, y, ids)
    first = (x.double() @ layer.router[0].double()) < 0       # then expert 7's score of zero is the largest
    for t in range(3):
        want = [7, 0, 1, 2, 3] if first[t] else [0, 1, 2, 3, 4]
        assert ids[t].tolist() == want


def test_nan_and_infinite_tokens_stay_alone():
    layer = Layer(6, 128, 32, 9, 3, abi.T_BF16, 64)
    x = torch.randn(6, 128, device="cuda").bfloat16()
    x[1, 3] = float("nan"); x[4] = float("inf")
    y = torch.empty_like(x); ids = torch.full((6, 3), -1, dtype=torch.int32, device="cuda"); w = torch.empty(6, 3, device="cuda")
    layer(x, y, ids, w)
    assert ((ids >= 0) & (ids < 9)).all()
    assert ids[1].tolist() == [0, 1, 2] and y[1].isnan().all()
    keep = [0, 2, 3, 5]
    layer.check(x[keep], y[keep], ids[keep], w[keep])


def test_large_hidden_values_in_f16():
    """hidden values past f16's range: the layer's output is what counts"""
    layer = Layer(8, 128, 64, 4, 2, abi.T_F16, 64)
    layer.down.s.view(torch.bfloat16).mul_(2.0 ** -14)
    layer.down.value *= 2.0 ** -14
    x = (100 * torch.randn(2, 128, device="cuda")).half()
    y = torch.empty_like(x)
    u = x.double() @ layer.up.value[0].t()
    assert (u.abs().max() ** 2) > 65504
    layer(x, y)
    assert y.isfinite().all()
    layer.check(x, y, None, None)


def test_streams_graphs_and_repeats():
    layer = Layer(10, 512, 256, 16, 4, abi.T_BF16, 128)
    x = torch.randn(7, 512, device="cuda").bfloat16()
    y, z = torch.empty_like(x), torch.empty_like(x)
    ws = layer(x, y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        layer(x, z, stream=torch.cuda.current_stream().cuda_stream, ws=ws)
    for _ in range(3):
        z.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, z)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()      # two at a time, each with its own workspace
    ya, yb, wb = torch.empty_like(x), torch.empty_like(x), torch.empty_like(ws)
    torch.cuda.synchronize()
    for _ in range(20):
        layer(x, ya, stream=a.cuda_stream, ws=ws)
        layer(x, yb, stream=b.cuda_stream, ws=wb)
    torch.cuda.synchronize()
    assert torch.equal(ya, y) and torch.equal(yb, y)
    assert V.lib().vela_device_error(1) == 0


@pytest.mark.parametrize("T,f32", [(1, False), (3, True), (20, False)])
def test_two_streams_at_a_time(T, f32):
    """both forms of the layer (few tokens with a router of their own type; else), on two streams with a workspace each"""
    layer = Layer(14, 256, 64, 12, 3, abi.T_BF16, 64, router_f32=f32)
    x = torch.randn(T, 256, device="cuda").bfloat16()
    y = torch.empty_like(x)
    wa = layer(x, y)
    layer.check(x, y, None, None)
    wb = torch.empty_like(wa)
    ya, yb = torch.empty_like(x), torch.empty_like(x)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        layer(x, ya, stream=a.cuda_stream, ws=wa)
        layer(x, yb, stream=b.cuda_stream, ws=wb)
    torch.cuda.synchronize()
    assert torch.equal(ya, y) and torch.equal(yb, y)
    assert V.lib().vela_device_error(1) == 0


def test_both_forms_agree():
    """a router in 32 bits takes the form with a barrier, the same numbers in bf16 the form for few tokens"""
    for T in (1, 4):
        layer = Layer(16, 384, 136, 9, 2, abi.T_BF16, 128)
        x = torch.randn(T, 384, device="cuda").bfloat16()
        out = []
        for f32 in (False, True):
            layer.router = layer.router.float() if f32 else layer.router
            y = torch.empty_like(x); ids = torch.empty(T, 2, dtype=torch.int32, device="cuda"); w = torch.empty(T, 2, device="cuda")
            layer(x, y, ids, w)
            layer.check(x, y, ids, w)
            out.append(ids)
        assert torch.equal(*out)


def test_no_tokens():
    layer = Layer(11, 64, 16, 2, 1, abi.T_BF16, 64)
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    c = layer.c()
    V.check(V.lib().vela_moe_w4(None, abi.T_BF16, None, 64, 0, ctypes.byref(c), None, 64, None, None, None, 0))


def test_wait_timeout_then_right():
    """the grid's barrier waits for a block that does not exist: the call ends by itself, reports, and leaves nothing behind"""
    layer = Layer(12, 256, 128, 8, 2, abi.T_BF16, 64)
    x = torch.randn(4, 256, device="cuda").bfloat16()
    y = torch.full_like(x, 7)
    c = layer.c()
    n = V.lib().vela_moe_w4_workspace(ctypes.byref(c), 4)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    assert V.lib().vela_device_error(1) == 0
    V.check(V.lib().vela_moe_w4_stalled(None, abi.T_BF16, ptr(x), 256, 4, ctypes.byref(c), ptr(y), 256, None, None, ptr(ws), n, 1_000_000))
    torch.cuda.synchronize()
    assert V.lib().vela_device_error(1) != 0 and (y == 7).all()
    layer(x, y, ws=ws)
    assert V.lib().vela_device_error(1) == 0
    layer.check(x, y, None, None)
