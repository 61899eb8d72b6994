"""Results of the operators under autograd may be changed in place, as torch's own: for inputs of any number of
dimensions, with and without gradients."""
import pytest

pytestmark = pytest.mark.gpu
SHAPES = [(20, 64), (3, 7, 64), (2, 1, 3, 64), (64,), (0, 64), (2, 0, 64)]


def _torch():
    import torch
    from neuroflow_b200 import ops
    return torch, ops


def _call(name, x, w, r):
    _, ops = _torch()
    if name == "linear":
        return ops.linear(x, w, act=1)
    if name == "linear with residual":
        return ops.linear(x, w, residual=r)
    if name == "fp8_linear":
        return ops.fp8_linear(x, w)
    if name == "layer_norm_autograd":
        return ops.layer_norm_autograd(x)
    return ops.rms_norm_autograd(x)


NAMES = ["linear", "linear with residual", "fp8_linear", "rms_norm_autograd", "layer_norm_autograd"]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("name", NAMES)
def test_in_place_after_the_call(name, shape):
    torch, _ = _torch()
    gen = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()
    x, w, r = rnd(*shape).requires_grad_(), rnd(48, 64).requires_grad_(), rnd(*shape[:-1], 48)
    y = _call(name, x, w, r)
    want = 2 * y.detach()
    dy = rnd(*y.shape)
    twice, = torch.autograd.grad(y, x, 2 * dy)  # (what dy gives for 2 y)
    y = _call(name, x, w, r)
    version = y._version
    y.mul_(2)
    assert torch.equal(y.detach(), want) and y._version == version + 1 and not y._is_view()
    got, = torch.autograd.grad(y, x, dy)
    assert got.shape == x.shape and torch.equal(got, twice)
    # made without gradients, added to with them
    p = rnd(*y.shape).requires_grad_()
    with torch.no_grad():
        y = _call(name, x, w, r)
    y.add_(p)
    assert torch.equal(torch.autograd.grad(y, p, dy)[0], dy)
    y = _call(name, x.detach(), w.detach(), r)
    y.add_(p)
    assert torch.equal(torch.autograd.grad(y, p, dy)[0], dy)

