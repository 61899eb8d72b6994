"""Gradients made under create_graph have memory of their own: changing one in place changes neither another gradient
nor what the caller gave to the backward pass."""
import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    from neuroflow_b200 import ops
    return torch, ops


def _all_apart(grads, given):
    """Each gradient is doubled in place; the others and `given` stay."""
    torch, _ = _torch()
    for i, g in enumerate(grads):
        rest = [t for j, t in enumerate((*grads, *given)) if j != i]
        before, want = [t.detach().clone() for t in rest], 2 * g.detach()
        with torch.no_grad():
            g.mul_(2)
        assert torch.equal(g.detach(), want) and all(torch.equal(t.detach(), b) for t, b in zip(rest, before)), i


@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("lead", [(20,), (3, 7), ()])
def test_linear(lead, act):
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()
    leaves = [rnd(*lead, 64).requires_grad_(), rnd(24, 64).requires_grad_(), rnd(24).requires_grad_(), rnd(*lead, 24).requires_grad_()]
    dy = rnd(*lead, 24)
    y = ops.linear(*leaves[:3], act=act, residual=leaves[3])
    plain = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    grads = torch.autograd.grad(y, leaves, dy, create_graph=True)
    assert all(torch.equal(p, g.detach()) for p, g in zip(plain, grads))
    _all_apart(grads, (dy,))


@pytest.mark.parametrize("stream", ["bfloat16", "float32"])
@pytest.mark.parametrize("used", ["both", "norm", "sum"])
@pytest.mark.parametrize("params", [True, False])
def test_rms_norm(stream, used, params):
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(2)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()
    x, h = rnd(9, 130).requires_grad_(), rnd(9, 130).to(getattr(torch, stream)).requires_grad_()
    g = rnd(130).requires_grad_() if params and used != "sum" else None
    n, s = ops.rms_norm_autograd(x, g, residual=h)
    outs = {"both": (n, s), "norm": (n,), "sum": (s,)}[used]
    given = tuple(rnd(9, 130).to(o.dtype) for o in outs)
    leaves = [t for t in (x, h, g) if t is not None]
    plain = torch.autograd.grad(outs, leaves, given, retain_graph=True)
    grads = torch.autograd.grad(outs, leaves, given, create_graph=True)
    assert all(torch.equal(p, q.detach()) for p, q in zip(plain, grads))
    _all_apart(grads, given)


def test_leaves_grads():
    """The same through backward(): .grad of the residual and of x."""
    torch, ops = _torch()
    x, h = (torch.randn(4, 64, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    n, s = ops.rms_norm_autograd(x, None, residual=h)
    dy = torch.ones_like(n)
    (n + s).backward(dy, create_graph=True)
    _all_apart((x.grad, h.grad), (dy,))
