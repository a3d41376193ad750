"""vela_gemv_w4 against the products in 64 bits: every activation and result type, group size and scale type, with and without
zero points, one to many rows, odd sizes, strides, and the fused bias and residual.

Bounds: 16-bit activations times integers are exact, 8-bit ones are summed in integers; what rounds is the 32-bit sum over
groups, bounded by the number of additions times the total magnitude (tests/lm_util.sum_bound), and Y's type once.
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

XT = [abi.T_BF16, abi.T_F16, abi.T_I8, abi.T_E4M3]
YT = [abi.T_F32, abi.T_BF16, abi.T_F16]


def make_x(gen, xt, M, K, xgroup, ld, off):
    """X [M, K], its scales or None, and its values in 64 bits"""
    x, _ = strided(M, K, ld, off, DT[xt])
    if xt in (abi.T_BF16, abi.T_F16):
        x.copy_(torch.randn(M, K, generator=gen, device="cuda"))
        return x, None, x.double()
    ng = -(-K // xgroup) if xgroup else 1
    scale = torch.rand(M, ng, generator=gen, device="cuda") + 0.1
    if xt == abi.T_I8:
        x.copy_(torch.randint(-127, 128, (M, K), generator=gen, device="cuda"))
    else:
        x.copy_((100 * torch.randn(M, K, generator=gen, device="cuda")).clamp(-448, 448).to(torch.float8_e4m3fn))
    v = x.to(torch.float32).double()
    return x, scale, v * scale.double().repeat_interleave(xgroup or K, 1)[:, :K]


def call(xt, x, scale, xgroup, M, W, bias, res, yt, y, stream=None, ldx=None):
    c = W.c()
    return V.lib().vela_gemv_w4(stream, xt, ptr(x), ldx or x.stride(0), ptr(scale), xgroup, M, ctypes.byref(c), ptr(bias), ptr(res),
                                res.stride(0) if res is not None else 0, yt, ptr(y), y.stride(0))


def check(xv, W, bias, res, yt, y):
    w = W.value[0]
    want = xv @ w.t()
    mass = xv.abs() @ w.abs().t()
    if bias is not None:
        want = want + bias.double(); mass = mass + bias.double().abs()
    if res is not None:
        want = want + res.double(); mass = mass + res.double().abs()
    # the zero points add to the integer sums before they cancel, so the magnitude counts codes, at most 15 a step
    within(y, want, sum_bound(W.K, mass) + want.abs() * ROUND[yt] + TINY[yt], "Y")


CASES = [
    # M, N, K
    (1, 1, 1), (1, 16, 64), (1, 17, 65), (2, 33, 96), (3, 100, 40), (1, 1024, 1024), (8, 48, 1000), (9, 50, 1280), (5, 2000, 130),
    (16, 129, 2048), (17, 64, 513), (31, 300, 192), (32, 1000, 256), (33, 40, 640), (70, 90, 128), (1, 5003, 333), (1, 31, 9000), (4, 4096, 4096),
]


@pytest.mark.parametrize("xt", XT)
@pytest.mark.parametrize("M,N,K", CASES)
def test_against_64_bits(xt, M, N, K):
    gen = torch.Generator(device="cuda"); gen.manual_seed(M * 7 + N * 11 + K * 13 + xt)
    scaled = xt in (abi.T_I8, abi.T_E4M3)
    for i, (group, zero) in enumerate([(32, False), (64, True), (128, False), (128, True), (32, True), (64, False)]):
        W = W4(N * K + i, N, K, group, zero, abi.T_F16 if i % 2 else abi.T_BF16)
        xgroup = (0, 64, 128)[i % 3] if scaled else 0
        yt = YT[i % 3]
        for layout in ("plain", "strided", "odd"):
            ld = {"plain": K, "strided": (K + 23) // 8 * 8, "odd": K + 3}[layout]
            x, scale, xv = make_x(gen, xt, M, K, xgroup, ld, 1 if layout == "odd" else 0)
            bias = torch.randn(N, generator=gen, device="cuda") if layout != "plain" else None
            res = torch.randn(M, N + 5, generator=gen, device="cuda").to(DT[yt])[:, :N] if layout == "strided" else None
            y, yb = strided(M, N, N + (0 if layout == "plain" else 3), 1 if layout == "odd" else 0, DT[yt])
            V.check(call(xt, x, scale, xgroup, M, W, bias, res, yt, y, ldx=ld))
            check(xv, W, bias, res, yt, y)
            off, ldy = (1 if layout == "odd" else 0), y.stride(0) if M > 1 else N + (0 if layout == "plain" else 3)
            idx = torch.arange(yb.numel(), device="cuda") - off
            inside = (idx >= 0) & (idx < M * ldy) & (idx % ldy < N)
            assert (yb.view(torch.uint8).view(yb.numel(), -1)[~inside] == 0x5A).all(), "written outside Y"


def test_residual_in_place():
    W = W4(3, 200, 320, 64, False, abi.T_BF16)
    x = torch.randn(4, 320, device="cuda").bfloat16()
    res = torch.randn(4, 200, device="cuda").bfloat16()
    y = res.clone()
    V.check(call(abi.T_BF16, x, None, 0, 4, W, None, y, abi.T_BF16, y))
    check(x.double(), W, None, res, abi.T_BF16, y)


def test_padding_of_the_layout_is_never_used():
    """codes, scales and zero points of rows past N and columns past K may hold anything, NaN scales included"""
    N, K, group = 21, 100, 32
    W = W4(5, N, K, group, True, abi.T_BF16)
    n, k = torch.arange(32, device="cuda")[:, None], torch.arange(128, device="cuda")[None, :]
    i = k % 64
    at = ((n // 16) * 2 + k // 64) * 512 + 16 * (4 * (n % 8) + i % 32 // 8) + 8 * (i // 32) + i % 8 // 4 * 4 + torch.tensor([0, 2, 1, 3], device="cuda")[i % 4]
    high = (n // 8 % 2).expand(32, 128)
    pad = (n >= N) | (k >= K)
    for nib in (0, 1):
        sel = at[pad & (high == nib)]
        W.q[sel] |= 0xF0 if nib else 0x0F
    rows = torch.arange(16, 32, device="cuda")
    s = W.s.view(torch.bfloat16).view(2, 4, 8, 2)
    for r in rows.tolist():
        if r >= N:
            s[1, :, r % 8, r // 8 % 2] = float("nan")
    for xt in XT:
        gen = torch.Generator(device="cuda"); gen.manual_seed(1)
        x, scale, xv = make_x(gen, xt, 3, K, 64 if xt >= abi.T_I8 else 0, K, 0)
        y = torch.empty(3, N, device="cuda")
        V.check(call(xt, x, scale, 64, 3, W, None, None, abi.T_F32, y))
        check(xv, W, None, None, abi.T_F32, y)


def test_nan_and_infinity_stay_in_their_row():
    W = W4(6, 40, 256, 128, False, abi.T_BF16)
    x = torch.randn(9, 256, device="cuda").bfloat16()
    x[2, 5] = float("nan"); x[8, 255] = float("inf")
    y = torch.empty(9, 40, device="cuda")
    V.check(call(abi.T_BF16, x, None, 0, 9, W, None, None, abi.T_F32, y))
    assert y[2].isnan().all() and not y[8].isfinite().any()
    keep = [0, 1, 3, 4, 5, 6, 7]
    check(x[keep].double(), W, None, None, abi.T_F32, y[keep])


def test_rows_do_not_depend_on_their_neighbours():
    """a row's result is the same, bit for bit, in a call of its own kind with other rows"""
    W = W4(7, 512, 2048, 128, False, abi.T_BF16)
    x = torch.randn(8, 2048, device="cuda").bfloat16()
    y = torch.empty(8, 512, device="cuda"); z = torch.empty(8, 512, device="cuda")
    V.check(call(abi.T_BF16, x, None, 0, 8, W, None, None, abi.T_F32, y))
    x2 = x.clone(); x2[1:] = 7
    V.check(call(abi.T_BF16, x2, None, 0, 8, W, None, None, abi.T_F32, z))
    assert torch.equal(y[0], z[0])


def test_streams_graphs_and_repeats():
    W = W4(8, 1000, 4096, 64, True, abi.T_F16)
    x = torch.randn(2, 4096, device="cuda").half()
    y = torch.empty(2, 1000, device="cuda"); z = torch.empty(2, 1000, device="cuda")
    V.check(call(abi.T_F16, x, None, 0, 2, W, None, None, abi.T_F32, y))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        V.check(call(abi.T_F16, x, None, 0, 2, W, None, None, abi.T_F32, z, stream=torch.cuda.current_stream().cuda_stream))
    for _ in range(3):
        z.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, z)


def test_offsets_beyond_32_bits():
    """a leading dimension that puts rows past 2^32 bytes: the rows of X and Y are found with 64-bit offsets"""
    W = W4(9, 48, 128, 128, False, abi.T_BF16)
    ld = (1 << 30) + 8
    x = torch.zeros(2 * ld + 128, dtype=torch.bfloat16, device="cuda").as_strided((3, 128), (ld, 1))
    x.copy_(torch.randn(3, 128, device="cuda"))
    y = torch.zeros(2 * ld + 48, dtype=torch.bfloat16, device="cuda").as_strided((3, 48), (ld, 1))
    V.check(call(abi.T_BF16, x, None, 0, 3, W, None, None, abi.T_BF16, y))
    check(x.double(), W, None, None, abi.T_BF16, y)


def test_no_rows():
    W = W4(1, 16, 64, 64, False, abi.T_BF16)
    c = W.c()
    V.check(V.lib().vela_gemv_w4(None, abi.T_BF16, None, 64, None, 0, 0, ctypes.byref(c), None, None, 0, abi.T_BF16, None, 16))


@pytest.mark.parametrize("xt", [abi.T_BF16, abi.T_I8])
def test_more_rows_than_a_grid_holds(xt):
    """65535 times 16 rows fit a grid; a call may have more"""
    M, N, K = 65535 * 16 + 21, 16, 32
    gen = torch.Generator(device="cuda"); gen.manual_seed(xt)
    W = W4(31, N, K, 32, True, abi.T_BF16)
    x, scale, xv = make_x(gen, xt, M, K, 0, K, 0)
    y = torch.full((M, N), float("nan"), device="cuda")
    res = torch.randn(M, N, generator=gen, device="cuda")
    V.check(call(xt, x, scale, 0, M, W, None, res, abi.T_F32, y))
    check(xv, W, None, res, abi.T_F32, y)
