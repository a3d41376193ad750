"""One decoding step between two attention calls, with weights in 4 bits: the residual's addition and norm to int8 rows, the attention's
output projection on them, the next addition and norm, and a mixture-of-experts layer.  Random weights; runs on one B200.

    python examples/decode_step.py [--tokens 4] [--width 1024] [--hidden 512] [--experts 16] [--topk 2]
"""
import argparse
import ctypes
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import vela_b200 as V  # noqa: E402
from vela_b200 import abi  # noqa: E402


def to_gpu(parts):
    """weights of w4_quantize (one, or the experts' one after another) on the GPU: (tensors to keep, abi.W4)"""
    q, s = (torch.from_numpy(np.concatenate([p[k] for p in parts]).view(np.uint8)).cuda() for k in ("q", "scale"))
    z = torch.from_numpy(np.concatenate([p["zero"] for p in parts])).cuda() if parts[0]["zero"] is not None else None
    p = parts[0]
    return (q, s, z), abi.W4(q.data_ptr(), s.data_ptr(), z.data_ptr() if z is not None else None, p["N"], p["K"], p["group"], p["scale_type"])


class Step:
    """Weights, buffers and the calls of one layer's feed-forward part."""

    def __init__(self, tokens, width, hidden, experts, topk, seed=0):
        r = np.random.default_rng(seed)
        self.T, self.D, self.E, self.k = tokens, width, experts, topk
        self.proj = r.normal(0, width ** -0.5, (width, width)).astype(np.float32)
        self.gate, self.up = (r.normal(0, width ** -0.5, (experts, hidden, width)).astype(np.float32) for _ in range(2))
        self.down = r.normal(0, hidden ** -0.5, (experts, width, hidden)).astype(np.float32)
        self.router = torch.from_numpy(r.normal(0, width ** -0.5, (experts, width)).astype(np.float32)).cuda().bfloat16()
        self.norms = [torch.from_numpy((1 + 0.1 * r.normal(0, 1, width)).astype(np.float32)).cuda().bfloat16() for _ in range(2)]
        self.packed = {"proj": [V.w4_quantize(self.proj, 128, asym=True)],
                       "up": [V.w4_quantize(V.moe_gate_up(g, u), 64) for g, u in zip(self.gate, self.up)],
                       "down": [V.w4_quantize(d, 64) for d in self.down]}
        (self.keep_proj, self.w_proj), (self.keep_up, w_up), (self.keep_down, w_down) = (to_gpu(self.packed[n]) for n in ("proj", "up", "down"))
        self.layer = abi.Moe(width, hidden, experts, topk, self.router.data_ptr(), abi.T_BF16, None, 0, 1, 1.0, w_up, w_down)
        empty = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
        self.s1, self.s2, self.a, self.n2, self.y = (empty(tokens, width) for _ in range(5))
        self.q, self.qscale = empty(tokens, width, dtype=torch.int8), empty(tokens, dtype=torch.float32)
        self.ids, self.w = empty(tokens, topk, dtype=torch.int32), empty(tokens, topk, dtype=torch.float32)
        n = V.lib().vela_moe_w4_workspace(ctypes.byref(self.layer), tokens)
        self.ws = empty(n, dtype=torch.uint8)

    def __call__(self, x, residual):
        """x: the attention's output; residual: the stream it is added to.  Returns the new residual stream and the experts' output."""
        L, T, D, stream = V.lib(), self.T, self.D, torch.cuda.current_stream().cuda_stream
        p = lambda t: t.data_ptr()  # noqa: E731
        # s1 = x + residual; q ~ norm(s1) in 8 bits with a scale a row
        V.check(L.vela_rms_norm_q8(stream, abi.T_BF16, p(x), D, p(residual), D, p(self.norms[0]), 1e-5, T, D, p(self.s1), D, None, 0,
                                   abi.T_I8, p(self.q), D, p(self.qscale), 0))
        V.check(L.vela_gemv_w4(stream, abi.T_I8, p(self.q), D, p(self.qscale), 0, T, ctypes.byref(self.w_proj), None, None, 0,
                               abi.T_BF16, p(self.a), D))
        # s2 = a + s1; n2 = norm(s2)
        V.check(L.vela_rms_norm_q8(stream, abi.T_BF16, p(self.a), D, p(self.s1), D, p(self.norms[1]), 1e-5, T, D, p(self.s2), D, p(self.n2), D,
                                   abi.T_I8, None, 0, None, 0))
        V.check(L.vela_moe_w4(stream, abi.T_BF16, p(self.n2), D, T, ctypes.byref(self.layer), p(self.y), D, p(self.ids), p(self.w), p(self.ws), self.ws.numel()))
        return self.s2, self.y


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("tokens", 4), ("width", 1024), ("hidden", 512), ("experts", 16), ("topk", 2)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args(argv)
    step = Step(a.tokens, a.width, a.hidden, a.experts, a.topk)
    x, residual = (torch.randn(a.tokens, a.width, device="cuda").bfloat16() for _ in range(2))
    step(x, residual)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):                      # the step as a server replays it
        step(x, residual)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for _ in range(10):
        graph.replay()
    begin.record()
    for _ in range(100):
        graph.replay()
    end.record()
    end.synchronize()
    print("tokens %d, width %d, %d experts of %d, top %d: %.1f us a step; experts of the first token: %s" % (
        a.tokens, a.width, a.experts, a.hidden, a.topk, begin.elapsed_time(end) * 10, step.ids[0].tolist()))


if __name__ == "__main__":
    main()
