"""vela_gemv_w4 in the forms that only many rows against many row tiles take (two row tiles a warp, three column tiles).  The bounds are those of tests/test_gemv_w4_gpu.py."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

import vela_b200 as V  # noqa: E402
from vela_b200 import abi  # noqa: E402
from tests.lm_util import DT, W4, strided  # noqa: E402
from tests.test_gemv_w4_gpu import XT, YT, call, check, make_x  # noqa: E402

CASES = [
    # M, N, K: more than 148 row tiles of 16, an even or odd number of them, one warp a row group or several
    (9, 2385, 200), (16, 2400, 100), (12, 2500, 2100), (16, 5003, 333), (25, 2400, 64), (27, 2400, 1000), (33, 4800, 130), (47, 2369, 577),
    # three column tiles, one of them partial or not
    (17, 2385, 1000), (20, 90, 2300), (24, 5003, 130),
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
        for layout in ("plain", "odd"):
            ld, off = (K, 0) if layout == "plain" else (K + 3, 1)
            x, scale, xv = make_x(gen, xt, M, K, xgroup, ld, off)
            bias = torch.randn(N, generator=gen, device="cuda") if layout == "odd" else None
            res = torch.randn(M, N, generator=gen, device="cuda").to(DT[yt]) if layout == "plain" else None
            ldy = N + 3 * off
            y, yb = strided(M, N, ldy, off, DT[yt])
            V.check(call(xt, x, scale, xgroup, M, W, bias, res, yt, y, ldx=ld))
            check(xv, W, bias, res, yt, y)
            idx = torch.arange(yb.numel(), device="cuda") - off
            inside = (idx >= 0) & (idx < M * ldy) & (idx % ldy < N)
            assert (yb.view(torch.uint8).view(yb.numel(), -1)[~inside] == 0x5A).all(), "written outside Y"
