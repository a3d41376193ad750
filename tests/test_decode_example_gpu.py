"""examples/decode_step.py: the operators run together as a user chains them, against the same chain in 64 bits on the quantised weights."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

import numpy as np  # noqa: E402

from examples.decode_step import Step, main  # noqa: E402
from tests.test_lmops_cpu import unpack  # noqa: E402


def value(p):
    codes, scales, zeros = unpack(p["q"], p["scale"], p["zero"], p["N"], p["K"], p["group"], p["scale_type"])
    rep = lambda a: np.repeat(a.astype(np.float64), p["group"], 1)[:, :p["K"]]  # noqa: E731
    return torch.from_numpy((codes - (rep(zeros) if zeros is not None else 8.0)) * rep(scales)).cuda()


def norm(h, g):
    return h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-5) * g.double()


@pytest.mark.parametrize("tokens", [1, 5])
def test_step_against_64_bits(tokens):
    """Every operator is held to its own bound elsewhere; here the chain is, to what its roundings leave: an int8 row (half a
    step of 1/127 of the row's largest value), four bf16 roundings of 2^-8, relative to the results' size."""
    s = Step(tokens, 192, 64, 6, 2, seed=tokens)
    gen = torch.Generator(device="cuda"); gen.manual_seed(tokens)
    x, r = (torch.randn(tokens, 192, generator=gen, device="cuda").bfloat16() for _ in range(2))
    s2, y = s(x, r)
    s1 = x.double() + r.double()
    want2 = norm(s1, s.norms[0]) @ value(s.packed["proj"][0]).t() + s1
    assert (s2.double() - want2).norm() <= 0.02 * want2.norm()
    n2 = norm(s2.double(), s.norms[1])                 # from the step's own sum on: the choice of experts is then the same
    p = torch.softmax(n2 @ s.router.double().t(), 1)
    assert torch.equal(s.ids.long(), torch.sort(p, dim=1, descending=True, stable=True).indices[:, :2])
    want = torch.zeros_like(n2)
    i = torch.arange(64, device="cuda")
    for t in range(tokens):
        w = p[t, s.ids[t].long()]
        for j, e in enumerate(s.ids[t].tolist()):
            u = value(s.packed["up"][e]) @ n2[t]
            gate, up = u[i // 8 * 16 + i % 8], u[i // 8 * 16 + i % 8 + 8]
            want[t] += w[j] / w.sum() * (value(s.packed["down"][e]) @ (gate * torch.sigmoid(gate) * up))
    assert (y.double() - want).norm() <= 0.02 * want.norm()


def test_command_line(capsys):
    main(["--tokens", "2", "--width", "256", "--hidden", "64", "--experts", "4"])
    assert "us a step" in capsys.readouterr().out
