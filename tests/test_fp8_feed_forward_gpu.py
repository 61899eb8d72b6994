"""The FP8 feed-forward example: layer norm, quantiser and product together, served and trained.

Tolerance.  An E4M3 code with a scale for 128 elements is off by at most 2^-4 of its value, 2^-4 / sqrt(3)
in the mean square at worst (errors uniform within a step).  A product of two such operands has the two
errors added in squares, and the sum over K keeps the ratio (independent signs): each layer adds at most
sqrt(2) 2^-4 / sqrt(3) = 0.051 of its own output.  The second layer's input carries the first layer's
error through GELU (slope at most 1.13): 0.051 * 1.13 + 0.051 = 0.109 of the branch, and bf16 roundings
2^-8; the residual x only lowers the ratio."""
import importlib.util
import os
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location("fp8_feed_forward", os.path.join(ROOT, "examples", "fp8_feed_forward.py"))
    m = importlib.util.module_from_spec(spec)
    sys.modules["fp8_feed_forward"] = m
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("tokens,dim,hidden", [(300, 256, 640), (65, 200, 333)])
def test_trains_and_serves(tokens, dim, hidden):
    ex = _example()
    losses, many, one = ex.run(tokens, dim, hidden, steps=8)
    assert losses[-1] < 0.8 * losses[0] and all(v == v for v in losses)
    assert many < 0.12 and one < 0.12


def test_gradients_follow_the_fp32_block():
    """The training form's gradients point where those of the fp32 block do: the FP8 operands add a
    relative error of at most 0.11 per product chain (see above), so the cosine stays above
    1 - 0.2^2 / 2 with two products' errors on each side."""
    import torch
    import torch.nn.functional as F
    ex = _example()
    torch.manual_seed(1)
    block = ex.FeedForward(256, 512)
    x = torch.randn(200, 256, device="cuda").bfloat16()
    dy = torch.randn(200, 256, device="cuda").bfloat16()
    block(x).backward(dy)
    got = [p.grad.clone() for p in block.parameters()]
    block.zero_grad(set_to_none=True)
    h = F.layer_norm(x.float(), (256,), block.gamma, block.beta)
    y = x.float() + F.gelu(h @ block.w1.t() + block.b1, approximate="tanh") @ block.w2.t() + block.b2
    y.backward(dy.float())
    for g, p in zip(got, block.parameters()):
        cos = torch.nn.functional.cosine_similarity(g.flatten().float(), p.grad.flatten(), dim=0)
        assert cos > 1 - 0.2 ** 2 / 2
