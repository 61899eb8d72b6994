"""What the differentiable operators do beyond a first backward pass: they refuse what they cannot do,
instead of leaving terms out."""
import pytest

pytestmark = pytest.mark.gpu


def _inputs():
    import torch
    from neuroflow_b200 import ops
    gen = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x, w, b, g = rnd(24, 160), rnd(48, 160) / 12, rnd(48), 1 + 0.1 * rnd(160)
    return torch, ops, x, w, b, g


def _forms(ops, w, b, g):
    return [lambda x: ops.fp8_linear(x, w, b), lambda x: ops.layer_norm_autograd(x, g, g)]


def test_second_derivatives_are_refused():
    """A gradient made under create_graph has no graph of its own: differentiating it is an error, and not a
    missing term.  What does not differentiate it works."""
    torch, ops, x, w, b, g = _inputs()
    from neuroflow_b200 import _nfx
    for t in (x, w, b, g):
        t.requires_grad_()
    for f, params in zip(_forms(ops, w, b, g), ((x, w, b), (x, g))):
        first = torch.autograd.grad((f(x) ** 2).sum(), params)
        for i in range(len(params)):
            y = f(x)
            grads = torch.autograd.grad((y ** 2).sum(), params, create_graph=True)
            assert all(torch.equal(p.detach(), q) for p, q in zip(grads, first))
            with pytest.raises(_nfx.NfxError) as ei:
                (y.sum() + (grads[i] ** 2).sum()).backward()
            assert ei.value.code == 1 and "second" in str(ei.value)
        y = f(x)
        torch.autograd.grad(y.sum(), params, create_graph=True)
        y.sum().backward()
        assert x.grad is not None
        x.grad = None


def test_gradients_made_under_create_graph_can_be_changed_in_place():
    torch, ops, x, w, b, g = _inputs()
    for t in (x, w, b, g):
        t.requires_grad_()
    for f, params in zip(_forms(ops, w, b, g), ((x, w, b), (x, g))):
        f(x).sum().backward(create_graph=True)
        for p in params:
            with torch.no_grad():
                p.grad.mul_(0.5)
                p.grad.zero_()
            p.grad = None


def test_forward_mode_is_refused():
    """A tangent would be dropped without a word; also where no gradient is asked for."""
    torch, ops, x, w, b, g = _inputs()
    from neuroflow_b200 import _nfx
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))
        calls = [lambda: ops.fp8_linear(dual(x), w, b), lambda: ops.fp8_linear(x, dual(w), b),
                 lambda: ops.fp8_linear(x, w, dual(b)), lambda: ops.layer_norm_autograd(dual(x), g),
                 lambda: ops.layer_norm_autograd(x, dual(g)), lambda: ops.layer_norm_autograd(x, g, dual(g))]
        for needs in (False, True):
            w.requires_grad_(needs), g.requires_grad_(needs)
            for grad in (True, False):
                with torch.set_grad_enabled(grad):
                    for i, call in enumerate(calls):
                        with pytest.raises(_nfx.NfxError) as ei:
                            call()
                        assert ei.value.code == 1 and "forward-mode" in str(ei.value), i
    w.requires_grad_(False)
    assert ops.fp8_linear(x, w, b).shape == (24, 48)


def _outs(ops, x, w, g):
    a, q = ops.fp8_quantise(x), ops.fp8_quantise(w, tile=True)
    return [((24, 160), lambda out: ops.layer_norm(x, g, out=out)), ((24, 48), lambda out: ops.fp8_gemm(a, q, out=out))]


def test_writing_into_out_is_seen_by_autograd():
    """A buffer that a backward pass has saved is changed: the backward pass says so."""
    torch, ops, x, w, b, g = _inputs()
    p = torch.ones((), device="cuda", requires_grad=True)
    for shape, call in _outs(ops, x, w, g):
        buf = torch.ones(shape, device="cuda")
        h = (buf * p).sum()
        version = buf._version
        assert call(buf) is buf
        assert buf._version > version
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            h.backward()
        with torch.inference_mode():
            call(torch.ones(shape, device="cuda"))
            inside = torch.ones(shape, device="cuda")
        call(inside)


def test_out_that_requires_grad_is_refused():
    torch, ops, x, w, b, g = _inputs()
    from neuroflow_b200 import _nfx
    for shape, call in _outs(ops, x, w, g):
        buf = torch.zeros(shape, device="cuda", requires_grad=True)
        with pytest.raises(_nfx.NfxError) as ei:
            call(buf)
        assert ei.value.code == 1 and "requires grad" in str(ei.value)
        torch.cuda.synchronize()
        assert not buf.detach().any()
        with torch.no_grad():
            call(buf)
        assert buf.detach().any()


def test_activation_numbers_are_not_cut_to_32_bits():
    torch, ops, x, w, b, g = _inputs()
    from neuroflow_b200 import _nfx
    a, q = ops.fp8_quantise(x), ops.fp8_quantise(w, tile=True)
    for act in (1 << 32, (1 << 32) + 1, -1, 3):
        with pytest.raises(_nfx.NfxError) as ei:
            ops.fp8_gemm(a, q, act=act)
        assert ei.value.code == 1


def test_out_may_be_x_but_not_a_part_of_its_memory():
    torch, ops, x, w, b, g = _inputs()
    from neuroflow_b200 import _nfx
    want = ops.layer_norm(x, g)
    hold = torch.empty(x.numel() + 160, device="cuda")
    xs, shifted = hold[:x.numel()].view_as(x), hold[160:].view_as(x)
    xs.copy_(x)
    with pytest.raises(_nfx.NfxError) as ei:
        ops.layer_norm(xs, g, out=shifted)
    assert ei.value.code == 1
    assert torch.equal(ops.layer_norm(xs, g, out=xs), want) and torch.equal(xs, want)
    # side by side in wider rows: no element is shared
    wide = torch.empty(24, 320, device="cuda")
    wide[:, :160] = x
    assert torch.equal(ops.layer_norm(wide[:, :160], g, out=wide[:, 160:]), want)
