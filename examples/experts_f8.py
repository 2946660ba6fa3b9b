"""A block of experts in e4m3 with scales per block of 128 on one GPU: as a server
runs it, and its router tuned while the experts stay as they are.

    python examples/experts_f8.py [tokens]

When a model is loaded, quantize_f8 turns its experts' weights into codes with a
scale per 128 x 128.  A block is then, beside the router's own product,

    q, s, h, v  = rms_norm_q8(x, norm, residual=h, fmt="e4m3_g128", normed=True)
    off, tok, p = expert_sort(ids, experts)         pairs (token, choice) by expert
    a           = f8_linear_experts(q, s, gate_up, ..., off, tok)
    q, s        = silu_mul_q8(a, fmt="e4m3_g128")
    y           = f8_linear_experts(q, s, down, ..., off)
    x           = expert_combine(y, p, w)           back to tokens, with weights

with no row gathered in memory and nothing read back by the host.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "qwen3.8-flash-next-fp4-local-spark_amd"))
import fp4x_kernels as F  # noqa: E402

FMT = "e4m3_g128"


class Rows(torch.autograd.Function):
    """Rows in the experts' order; their gradients are summed per token."""

    @staticmethod
    def forward(ctx, x, tokens, slots):
        ctx.save_for_backward(slots)
        return F.expert_rows(x, tokens)

    @staticmethod
    def backward(ctx, dy):
        return F.expert_combine(dy, *ctx.saved_tensors), None, None


class Combine(torch.autograd.Function):
    """The experts' rows back to their tokens, weighted; gradients of both."""

    @staticmethod
    def forward(ctx, y, slots, tokens, weights):
        ctx.save_for_backward(y, slots, weights, tokens)
        return F.expert_combine(y, slots, weights)

    @staticmethod
    def backward(ctx, dout):
        dy, dw = F.expert_combine_grad(dout, *ctx.saved_tensors)
        return dy, None, None, dw


class Experts:
    """norm -> router -> gate and up -> silu(gate) * up -> down -> weighted sum."""

    def __init__(self, norm, router, gate_up, down, picks, eps=1e-6):
        self.norm, self.router, self.picks, self.eps = norm, router, picks, eps
        self.gate_up, self.down = F.quantize_f8(gate_up), F.quantize_f8(down)

    def route(self, v):
        return torch.softmax(v.float() @ self.router.t(), -1).topk(self.picks, -1)

    def experts(self, q, s, ids):
        offsets, tokens, slots = F.expert_sort(ids, self.router.shape[0])
        a = F.f8_linear_experts(q, s, *self.gate_up, offsets, tokens)
        return F.f8_linear_experts(*F.silu_mul_q8(a, fmt=FMT), *self.down, offsets), tokens, slots

    def __call__(self, x, residual):
        """(output of the block, the next residual)"""
        q, s, residual, v = F.rms_norm_q8(x, self.norm, eps=self.eps, residual=residual, fmt=FMT, normed=True)
        w, ids = self.route(v)
        y, _, slots = self.experts(q, s, ids)
        return F.expert_combine(y, slots, w), residual

    def tune(self, x, target, steps, rate=0.5):
        """Steps of the router towards the target, through the frozen experts; the losses."""
        q, s, v = F.rms_norm_q8(x, self.norm, eps=self.eps, fmt=FMT, normed=True)
        self.router.requires_grad_()
        losses = []
        for _ in range(steps):
            w, ids = self.route(v)
            y, tokens, slots = self.experts(q, s, ids.detach())
            loss = (Combine.apply(y, slots, tokens, w).float() - target).square().mean()
            (grad,) = torch.autograd.grad(loss, self.router)
            with torch.no_grad():
                self.router -= rate * grad
            losses.append(float(loss.detach()))
        self.router.requires_grad_(False)
        return losses


def reference(x, residual, norm, router, gate_up, down, picks, eps=1e-6):
    """The same block in fp32 from the weights as they were."""
    h = (x.float() + residual.float()).to(residual.dtype)
    v = h.float() * torch.rsqrt(h.float().square().mean(-1, keepdim=True) + eps) * norm.float()
    w, ids = torch.softmax(v.to(x.dtype).float() @ router.t(), -1).topk(picks, -1)
    out = torch.zeros_like(v)
    for e in range(router.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        gate, up = (v[t] @ gate_up[e].float().t()).chunk(2, -1)
        out.index_add_(0, t, w[t, j][:, None] * ((torch.nn.functional.silu(gate) * up) @ down[e].float().t()))
    return out, h


def make(tokens, hidden=2560, inner=640, experts=16, seed=0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda") * scale
    weights = ((1 + 0.1 * r(hidden)).to(dtype), r(experts, hidden, scale=hidden ** -0.5),
               r(experts, 2 * inner, hidden, scale=0.02).to(dtype), r(experts, hidden, inner, scale=0.02).to(dtype))
    return weights, r(tokens, hidden).to(dtype), r(tokens, hidden, scale=2.0).to(dtype)


def main(tokens=1024, picks=4, **sizes):
    weights, x, residual = make(tokens, **sizes)
    block = Experts(*weights, picks)
    y, h = block(x, residual)
    want, h32 = reference(x, residual, *weights, picks)
    err = float((y.float() - want).norm() / want.norm())
    print(f"{tokens} tokens: relative error {err:.4f} against fp32 weights and activations, residual equal: "
          f"{bool(torch.equal(h, h32))}")

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yg, _ = block(x, residual)
    graph.replay()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(50):
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    print(f"{start.elapsed_time(end) * 20:.1f} us per block, replay equal: {bool(torch.equal(yg, y))}")

    losses = block.tune(x, want, 5)
    print("router's losses:", " ".join(f"{v:.5f}" for v in losses))
    return err


if __name__ == "__main__":
    main(*(int(a) for a in sys.argv[1:2]))
