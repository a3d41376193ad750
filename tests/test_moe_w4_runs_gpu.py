"""vela_moe_w4 on the forms that small layers do not reach: long and wide runs of the streaming loop (tests/moe_runs.py), hidden values past
f16's range in it, graphs and streams of the form with a barrier, and the few-token kernels with many experts and with 32 warps on a
row tile.  The bounds are those of tests/test_moe_w4_gpu.py.
"""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

import vela_b200 as V  # noqa: E402
from vela_b200 import abi  # noqa: E402
from tests.lm_util import DT, within  # noqa: E402
from tests.moe_runs import RUNS  # noqa: E402
from tests.test_moe_w4_gpu import Layer  # noqa: E402


def tokens(T, D, type, seed=1):
    return torch.randn(T, D, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(DT[type])


def run_and_check(layer, x):
    T = x.shape[0]
    y = torch.empty_like(x)
    ids = torch.full((T, layer.k), -1, dtype=torch.int32, device="cuda"); w = torch.full((T, layer.k), float("nan"), device="cuda")
    layer(x, y, ids, w)
    layer.check(x, y, ids, w)
    assert V.lib().vela_device_error(1) == 0
    return y


def within_type(got, want, bound, what=""):
    """what f16 cannot hold is stored as an infinity of its sign; the rest is within its bound"""
    if got.dtype == torch.float16:
        beyond = want.abs() - bound > 65520             # rounds to an infinity, whatever the error
        assert (got[beyond].double() == want[beyond].sign() * torch.inf).all()
        keep = want.abs() + bound < 65504
        got, want, bound = got[keep], want[keep], bound[keep]
        assert got.numel() > 0
    within(got, want, bound, what)


@pytest.mark.parametrize("T,D,I,E,k,type,group,zero", [r[0] for r in RUNS])
def test_runs(monkeypatch, T, D, I, E, k, type, group, zero):
    monkeypatch.setattr("tests.test_moe_w4_gpu.within", within_type)
    run_and_check(Layer(T + D + I + E, D, I, E, k, type, group, zero), tokens(T, D, type))


@pytest.mark.parametrize("T,D,I,E,k,type,group,zero", [
    (1, 256, 1288, 4, 2, abi.T_BF16, 128, False),      # 22 units of hidden columns for each of 16 row tiles
    (3, 200, 392, 8, 6, abi.T_F16, 32, True),          # 24 for each of 39, the last with 8 rows
    (2, 264, 648, 5, 3, abi.T_BF16, 64, True),         # 18 for each of 34
])
def test_few_tokens_of_few_row_tiles(T, D, I, E, k, type, group, zero):
    run_and_check(Layer(T * D + I, D, I, E, k, type, group, zero), tokens(T, D, type))


@pytest.mark.parametrize("T,E,k,type,score", [(1, 65, 8, abi.T_BF16, 0), (3, 100, 5, abi.T_F16, 1), (8, 128, 4, abi.T_BF16, 0), (2, 128, 16, abi.T_F16, 0), (5, 81, 6, abi.T_BF16, 1)])
def test_few_tokens_of_many_experts(T, E, k, type, score):
    run_and_check(Layer(T * E, 136, 16, E, k, type, 64, E % 2 == 0, score, bias=score == 1), tokens(T, 136, type))


@pytest.mark.parametrize("T", [2, 20])
def test_hidden_values_past_f16(T):
    """in 32 bits between the phases of the larger form, scaled by a power of two for its products"""
    layer = Layer(8, 128, 64, 4, 2, abi.T_F16, 64, router_f32=T == 2)
    layer.down.s.view(torch.bfloat16).mul_(2.0 ** -14)
    layer.down.value *= 2.0 ** -14
    x = (100 * tokens(T, 128, abi.T_F32)).half()
    assert ((x.double() @ layer.up.value[0].t()).abs().max() ** 2) > 65504
    assert run_and_check(layer, x).isfinite().all()


@pytest.mark.parametrize("T,f32", [(7, True), (20, False), (45, False)])
def test_graphs_and_streams_of_the_form_with_a_barrier(T, f32):
    """45 tokens: two cooperative kernels in one graph"""
    layer = Layer(10, 512, 256, 16, 4, abi.T_BF16, 128, router_f32=f32)
    x = tokens(T, 512, abi.T_BF16)
    y = run_and_check(layer, x)
    z = torch.empty_like(x)
    ws = layer(x, z)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        layer(x, z, stream=torch.cuda.current_stream().cuda_stream, ws=ws)
    for _ in range(3):
        z.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, z)
    assert V.lib().vela_device_error(1) == 0
