"""A token mixer's feed-forward block in FP8, served and trained with neuroflow_b200.ops.

    y = x + W2 gelu(W1 layer_norm(x) + b1) + b2

    python examples/fp8_feed_forward.py [--tokens 4096] [--dim 1024] [--hidden 4096] [--steps 20]

Serving: the weights are quantised once; a call is a layer norm straight into FP8, a product with
bias and GELU in its epilogue, a quantiser and a second product.  The same block answers a single
token.  Training: the same layers under autograd, bf16 activations and fp32 master weights, on a
synthetic regression target; the quantised block is then served.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from neuroflow_b200 import ops  # noqa: E402


class FeedForward(torch.nn.Module):
    """The block's parameters (fp32) and its training form."""

    def __init__(self, dim, hidden, device="cuda"):
        super().__init__()
        p = lambda t: torch.nn.Parameter(t.to(device))
        self.gamma, self.beta = p(torch.ones(dim)), p(torch.zeros(dim))
        self.w1, self.b1 = p(torch.randn(hidden, dim) / dim ** 0.5), p(torch.zeros(hidden))
        self.w2, self.b2 = p(torch.randn(dim, hidden) / hidden ** 0.5), p(torch.zeros(dim))

    def forward(self, x):
        h = ops.layer_norm_autograd(x, self.gamma, self.beta)
        h = F.gelu(ops.fp8_linear(h, self.w1, self.b1), approximate="tanh")
        return x + ops.fp8_linear(h, self.w2, self.b2)


class Served:
    """The block with its weights in FP8."""

    def __init__(self, block):
        with torch.no_grad():
            self.gamma, self.beta, self.b1, self.b2 = (t.detach().clone() for t in (block.gamma, block.beta, block.b1, block.b2))
            self.w1, self.w2 = ops.fp8_quantise(block.w1, tile=True), ops.fp8_quantise(block.w2, tile=True)

    def __call__(self, x):
        x8 = ops.layer_norm_fp8(x, self.gamma, self.beta)
        h = ops.fp8_gemm(x8, self.w1, bias=self.b1, act=1, out_dtype=x.dtype)
        return x + ops.fp8_gemm(ops.fp8_quantise(h), self.w2, bias=self.b2, out_dtype=x.dtype)


def plain(block, x):
    """The block in fp32, without FP8."""
    with torch.no_grad():
        h = F.layer_norm(x.float(), (x.shape[-1],), block.gamma, block.beta)
        h = F.gelu(h @ block.w1.t() + block.b1, approximate="tanh")
        return x.float() + h @ block.w2.t() + block.b2


def train(block, x, target, steps, lr):
    """Losses of `steps` Adam steps on the mean squared error."""
    opt = torch.optim.Adam(block.parameters(), lr=lr)
    losses = []
    for _ in range(steps):
        opt.zero_grad(set_to_none=True)
        loss = F.mse_loss(block(x).float(), target)
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return [float(v) for v in torch.stack(losses)]


def run(tokens, dim, hidden, steps, seed=0):
    """(losses of training, relative error of the served block against fp32 for all tokens and for one)."""
    torch.manual_seed(seed)
    block, teacher = FeedForward(dim, hidden), FeedForward(dim, hidden)
    x = torch.randn(tokens, dim, device="cuda").bfloat16()
    losses = train(block, x, plain(teacher, x), steps, lr=3e-3)
    served = Served(block)
    want = plain(block, x)
    rel = lambda a, b: float((a.float() - b).norm() / b.norm())
    return losses, rel(served(x), want), rel(served(x[:1]), want[:1])


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=4096)
    ap.add_argument("--dim", type=int, default=1024)
    ap.add_argument("--hidden", type=int, default=4096)
    ap.add_argument("--steps", type=int, default=20)
    a = ap.parse_args()
    losses, many, one = run(a.tokens, a.dim, a.hidden, a.steps)
    print(f"training: loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps")
    print(f"served in FP8 against fp32: relative error {many:.4f} ({a.tokens} tokens), {one:.4f} (one token)")
    served = Served(FeedForward(a.dim, a.hidden))
    for m in (1, a.tokens):
        x = torch.randn(m, a.dim, device="cuda").bfloat16()
        for _ in range(5):
            served(x)
        t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        t0.record()
        for _ in range(50):
            served(x)
        t1.record()
        torch.cuda.synchronize()
        print(f"served: {m} token(s) in {t0.elapsed_time(t1) / 50 * 1e3:.1f} us")


if __name__ == "__main__":
    main()
