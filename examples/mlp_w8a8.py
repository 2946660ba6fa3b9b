"""A gated MLP block in 8 bits on one GPU, as a server would run it.

    python examples/mlp_w8a8.py [tokens]

When a model is loaded, quantize_q8 turns its weights into int8 rows with a
scale per output channel.  A block is then four launches:

    q, s, h = rms_norm_q8(x, norm, residual=h)      norm, residual, int8 codes
    gu      = w8a8_linear(q, s, gate_up, ...)       one product for both halves
    q, s    = silu_mul_q8(gu)                       gate, int8 codes
    x       = w8a8_linear(q, s, down, ...)

and nothing that is wider than a layer's activations is written in between.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "qwen3.8-flash-next-fp4-local-spark_amd"))
import fp4x_kernels as F  # noqa: E402


class GatedMLP:
    """norm -> gate and up -> silu(gate) * up -> down, weights held in int8."""

    def __init__(self, norm, gate, up, down, eps=1e-6):
        self.norm, self.eps = norm, eps
        self.gate_up = F.quantize_q8(torch.cat([gate, up]))
        self.down = F.quantize_q8(down)

    def __call__(self, x, residual):
        """(output of the block, the next residual)"""
        q, s, residual = F.rms_norm_q8(x, self.norm, eps=self.eps, residual=residual)
        gu = F.w8a8_linear(q, s, *self.gate_up, out_dtype=x.dtype)
        return F.w8a8_linear(*F.silu_mul_q8(gu), *self.down, out_dtype=x.dtype), residual


def reference(x, residual, norm, gate, up, down, eps=1e-6):
    """The same block in fp32 from the weights as they were."""
    h = (x.float() + residual.float()).to(residual.dtype)
    v = h.float() * torch.rsqrt(h.float().square().mean(-1, keepdim=True) + eps) * norm.float()
    a = torch.nn.functional.silu(v @ gate.float().t()) * (v @ up.float().t())
    return a @ down.float().t(), h


def make(tokens, hidden=2560, inner=640, seed=0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)
    weights = ((1 + 0.1 * torch.randn(hidden, generator=g, device="cuda")).to(dtype), r(inner, hidden, scale=0.02),
               r(inner, hidden, scale=0.02), r(hidden, inner, scale=0.02))
    return weights, r(tokens, hidden), r(tokens, hidden, scale=2.0)


def main(tokens=1024):
    weights, x, residual = make(tokens)
    block = GatedMLP(*weights)
    y, h = block(x, residual)
    want, h32 = reference(x, residual, *weights)
    err = float((y.float() - want).norm() / want.norm())
    print(f"{tokens} tokens: relative error {err:.4f} against fp32 weights and activations, residual equal: "
          f"{bool(torch.equal(h, h32))}")

    # a step that is replayed: eight blocks captured once, new inputs copied in
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yg, hg = block(x, residual)
        yn, hn = yg, hg
        for _ in range(7):
            yn, hn = block(yn, hn)
    graph.replay()
    torch.cuda.synchronize()
    print(f"graph replay equal: {bool(torch.equal(yg, y) and torch.equal(hg, h))}")

    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(50):
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    print(f"{start.elapsed_time(end) * 1000 / 400:.1f} us per block")
    return err


if __name__ == "__main__":
    main(*(int(a) for a in sys.argv[1:2]))
