"""Routing of vela_moe_w4 where scores are not numbers, or probabilities equal or vanish in 32 bits, in both forms of the layer
(tests/test_moe_w4_gpu.py has the bounds; a router of 32 bits or more than 8 tokens take the form with a routing kernel of its own).
"""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from vela_b200 import abi  # noqa: E402
from tests.lm_util import sum_bound  # noqa: E402
from tests.test_moe_w4_gpu import Layer  # noqa: E402

FORMS = [(3, False), (3, True), (20, False)]       # tokens, router in 32 bits: the form for few tokens, the other one twice


def run(layer, x):
    T = x.shape[0]
    y = torch.empty_like(x)
    ids = torch.full((T, layer.k), -1, dtype=torch.int32, device="cuda"); w = torch.empty(T, layer.k, device="cuda")
    layer(x, y, ids, w)
    torch.cuda.synchronize()
    return y, ids, w


@pytest.mark.parametrize("T,f32", FORMS)
@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("bias", [False, True])
def test_a_nan_score_comes_last(T, f32, score, bias):
    """a router row of NaN: the other experts are scored, chosen and weighed as if it were not there"""
    layer = Layer(21, 128, 32, 9, 3, abi.T_BF16, 64, score=score, bias=bias, router_f32=f32)
    x = torch.randn(T, 128, generator=torch.Generator(device="cuda").manual_seed(T), device="cuda").bfloat16()
    layer.router[4] = float("nan")
    y, ids, w = run(layer, x)
    assert (ids != 4).all()
    layer.router[4] = 0                            # for the check: an expert that is out of the softmax's sum and of the choice
    rel = layer.route(x.double())[1]
    z = x.double() @ layer.router.double().t()
    z[:, 4] = -torch.inf
    p = torch.softmax(z, 1) if score == 0 else torch.sigmoid(z)
    pick = p if layer.bias is None else p + layer.bias.double()
    pick[:, 4] = -torch.inf
    layer.route = lambda _: (p, rel, pick)
    layer.check(x, y, ids, w)


@pytest.mark.parametrize("T,f32", FORMS)
@pytest.mark.parametrize("score", [0, 1])
def test_a_nan_expert_that_has_to_be_chosen(T, f32, score):
    """topk = E: the NaN comes last, with a NaN weight"""
    layer = Layer(22, 64, 16, 5, 5, abi.T_BF16, 64, score=score, renorm=0, router_f32=f32)
    x = torch.randn(T, 64, device="cuda").bfloat16()
    layer.router[2] = float("nan")
    _, ids, w = run(layer, x)
    assert (ids[:, 4] == 2).all() and w[:, 4].isnan().all() and w[:, :4].isfinite().all()
    assert all(sorted(r) == [0, 1, 2, 3, 4] for r in ids.tolist())


@pytest.mark.parametrize("T,f32", FORMS)
@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("top", [30.0, -130.0])
def test_choice_between_probabilities_that_are_equal_in_32_bits(T, f32, score, top):
    """Without a selection bias the order of the probabilities is that of the scores, also where they are all 1 or all 0 in 32 bits.  The scores
    rise with the expert's number, by about 3 from one to the next."""
    layer = Layer(24, 64, 16, 8, 3, abi.T_BF16, 64, score=score, renorm=0, router_f32=f32)
    x = torch.randn(T, 64, generator=torch.Generator(device="cuda").manual_seed(T), device="cuda").bfloat16()
    x[:, 0] = 1
    layer.router *= 0.05
    layer.router[:, 0] = (top + 3.0 * torch.arange(8, device="cuda")).to(layer.router.dtype)
    if score == 0:                                 # one expert far above: the others' probabilities vanish
        layer.router[3, 0] = top + 200
    z = x.double() @ layer.router.double().t()
    order = torch.sort(z, dim=1, descending=True, stable=True)
    gap = (order.values[:, :-1] - order.values[:, 1:]).amin()
    assert gap > 2 * sum_bound(64, x.double().abs() @ layer.router.double().abs().t()).amax()
    _, ids, w = run(layer, x)
    assert torch.equal(ids.long(), order.indices[:, :3])
    p = torch.softmax(z, 1) if score == 0 else torch.sigmoid(z)
    assert ((w.double() - p.gather(1, ids.long())).abs() <= 1e-3 * p.gather(1, ids.long()) + 2.0 ** -126).all()


@pytest.mark.parametrize("T,f32", FORMS)
@pytest.mark.parametrize("score", [0, 1])
def test_a_nan_comes_after_masked_experts(T, f32, score):
    layer = Layer(25, 64, 16, 5, 5, abi.T_BF16, 64, score=score, renorm=0, bias=True, router_f32=f32)
    x = torch.randn(T, 64, generator=torch.Generator(device="cuda").manual_seed(T), device="cuda").bfloat16()
    layer.router[2] = float("nan"); layer.bias[3] = -torch.inf
    _, ids, w = run(layer, x)
    assert (ids[:, 3] == 3).all() and (ids[:, 4] == 2).all()
    assert w[:, :4].isfinite().all() and w[:, 4].isnan().all()


@pytest.mark.parametrize("T,f32", FORMS)
@pytest.mark.parametrize("score", [0, 1])
def test_weights_of_vanishing_probabilities_sum_to_one(T, f32, score):
    """The chosen experts' probabilities are below the smallest float; divided by their sum they are ordinary numbers.  Sigmoid: every score is
    about -120 and less.  Softmax: the selection bias keeps the one expert out whose probability is not zero."""
    layer = Layer(23, 64, 16, 6, 3, abi.T_BF16, 64, score=score, bias=True, router_f32=f32)
    x = torch.randn(T, 64, generator=torch.Generator(device="cuda").manual_seed(T), device="cuda").bfloat16()
    x[:, 0] = 1
    layer.router *= 0.25
    layer.router[:, 0] = (-120 - 3.0 * torch.arange(6, device="cuda")).to(layer.router.dtype)
    layer.bias[:] = torch.tensor([3.0, 2.5, 2.0, -9.0, -9.0, -9.0], device="cuda")
    if score == 0:
        layer.router[5, 0] = 40.0
    p, _, _ = layer.route(x.double())
    assert (p[:, :3] < 2.0 ** -150).all() and (p[:, :3] > 0).all()
    y, ids, w = run(layer, x)
    assert w.isfinite().all() and (w.sum(1) - 1).abs().max() < 1e-5
    layer.check(x, y, ids, w)
