"""Layer norm (neuroflow_b200.ops / nfx_layer_norm*) against its formula in 64 bits.

Tolerances.  eps = 2^-24 is the fp32 unit roundoff.  A row's sums are formed by threads that add
at most d / 32 elements one after another and then join in a tree, so a sum of terms t is off by at
most (d / 32 + 16) eps sum |t|.  With n = d / 32 + 16:
  mean:  n eps mean|x|
  y:     the centred value is off by that much, the statistics' relative error is at most 2 n eps, a
         few roundings follow: |g| r (2 n eps max|x|) + 4 n eps |g xh| + 4 eps |b|, plus half an ulp
         of the output type.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
EPS32 = 2.0 ** -24
ULP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
EPS = 1e-5


def _torch():
    import torch
    from neuroflow_b200 import ops
    return torch, ops


def _case(rows, d, dtype, ptype, seed, offset=0.5):
    torch, _ = _torch()
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x = (rnd(rows, d) * torch.exp(0.5 * rnd(1, d)) + offset).to(dtype)
    return x, (1 + 0.2 * rnd(d)).to(ptype), (0.3 * rnd(d)).to(ptype), (0.1 * rnd(rows, d)).to(dtype)


def _plain(x, g, b, eps=EPS):
    x, g, b = x.double(), g.double(), b.double()
    mu = x.mean(1, keepdim=True)
    r = 1 / ((x - mu).square().mean(1, keepdim=True) + eps).sqrt()
    xh = (x - mu) * r
    return xh * g + b, mu, r, xh


def _y_tol(x, g, b, r, xh, dtype):
    n = x.shape[1] / 32 + 16
    x, g, b = x.double(), g.double(), b.double()
    y = xh * g + b
    t = g.abs() * r * (2 * n * EPS32 * x.abs().amax(1, keepdim=True)) + 4 * n * EPS32 * (g * xh).abs() + 4 * EPS32 * b.abs()
    tiny = 2.0 ** -25 if dtype == "float16" else 1e-38
    return t + ULP[dtype] * (y.abs() + t) + tiny


WIDTHS = [1, 2, 3, 31, 64, 66, 127, 128, 129, 256, 511, 514, 771, 1024, 1030, 1032, 2048, 2050, 4096, 4098, 5000, 8192, 9998,
          16384, 20001]


@pytest.mark.parametrize("dtype,ptype", [("float32", "float32"), ("bfloat16", "bfloat16"),
                                         ("bfloat16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("d", WIDTHS)
def test_forward(d, dtype, ptype):
    torch, ops = _torch()
    for rows in (1, 3, 130):
        x, g, b, _ = _case(rows, d, getattr(torch, dtype), getattr(torch, ptype), d + rows)
        y, mean, rstd = ops.layer_norm(x, g, b, EPS, stats=True)
        want, mu, r, xh = _plain(x, g, b)
        n = d / 32 + 16
        assert (mean.double() - mu[:, 0]).abs().le(n * EPS32 * x.double().abs().mean(1) + 1e-38).all()
        # the variance's relative error: 2 n eps, and the centred values' error against the spread
        spread = 2 * n * EPS32 * x.double().abs().amax(1) * r[:, 0]
        assert ((rstd.double() / r[:, 0] - 1).abs() <= 4 * n * EPS32 + 2 * spread).all()
        tol = _y_tol(x, g, b, r, xh, dtype) + (xh * g.double()).abs() * 2 * spread[:, None]
        assert ((y.double() - want).abs() <= tol).all(), (rows, d)
        y2 = ops.layer_norm(x, g, b, EPS)
        assert torch.equal(y, y2)


def test_no_parameters_and_leading_dimensions():
    torch, ops = _torch()
    x, _, _, _ = _case(12, 200, torch.float32, torch.float32, 1)
    one, zero = torch.ones(200, device="cuda"), torch.zeros(200, device="cuda")
    y = ops.layer_norm(x.view(2, 3, 2, 200))
    assert y.shape == (2, 3, 2, 200)
    assert torch.equal(y.view(12, 200), ops.layer_norm(x, one, zero))
    assert torch.equal(ops.layer_norm(x, one), ops.layer_norm(x, None, zero))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d,pitch,shift", [(256, 300, 0), (256, 256, 1), (1000, 1008, 8), (130, 133, 3), (4096, 4104, 2)])
def test_strides_and_alignment(dtype, d, pitch, shift):
    """Rows that start anywhere give what the same rows give when they are contiguous, to rounding,
    in the input, the gradient and the output; what lies between the rows is not written."""
    torch, ops = _torch()
    rows, dt = 37, getattr(torch, dtype)
    x, g, b, dy = _case(rows, d, dt, dt, 7)
    hold = torch.full((2, rows * pitch + 64,), 77.0, device="cuda", dtype=dt)
    place = lambda i: hold[i, shift:shift + rows * pitch].view(rows, pitch)[:, :d]
    xs, out = place(0), place(1)
    xs.copy_(x)
    y = ops.layer_norm(xs, g, b, EPS, out=out)
    assert y is out
    want, _, r, xh = _plain(x, g, b)
    n = d / 32 + 16
    spread = 2 * n * EPS32 * x.double().abs().amax(1, keepdim=True) * r
    tol = _y_tol(x, g, b, r, xh, dtype) + (xh * g.double()).abs() * 2 * spread
    assert ((y.double() - want).abs() <= tol).all()
    gap = hold[1, shift:shift + rows * pitch].view(rows, pitch)[:, d:]
    assert (gap == 77).all() and (hold[1, :shift] == 77).all()
    q = ops.layer_norm_fp8(xs, g, b, EPS)
    assert ((q.dequantise().double() - want).abs() <= want.abs() / 16 + q.scales.double().repeat_interleave(128, 1)[:, :d] * 2.0 ** -9 + tol).all()
    _, mean, rstd = ops.layer_norm(x, g, b, EPS, stats=True)
    dys = place(1)
    dys.copy_(dy)
    dx, dg, db = ops.layer_norm_backward(dys, xs, mean, rstd, g)
    _check_grad(dx, dg, db, dy, x, mean, rstd, g, dtype)


def test_rows_that_go_wrong_stay_alone():
    """A constant row gives beta; a row with an infinity or NaN gives NaN, and no other row does."""
    torch, ops = _torch()
    for d in (100, 1024, 5000):
        x, g, b, dy = _case(6, d, torch.float32, torch.float32, 3)
        x[1] = 4.25
        x[2, d // 2] = float("inf")
        x[4, 0] = float("nan")
        y, mean, rstd = ops.layer_norm(x, g, b, EPS, stats=True)
        assert torch.equal(y[1], b)
        assert y[2].isnan().all() and y[4].isnan().all()
        ok = [0, 1, 3, 5]
        assert y[ok].isfinite().all()
        assert torch.equal(y[ok], ops.layer_norm(x[ok], g, b, EPS))
        dx, _, _ = ops.layer_norm_backward(dy, x, mean, rstd, g)
        assert dx[ok].isfinite().all()
        q = ops.layer_norm_fp8(x, g, b, EPS)
        assert q.dequantise()[2].isnan().all() and q.dequantise()[ok].isfinite().all()


def test_large_mean_keeps_the_variance():
    torch, ops = _torch()
    x, g, b, _ = _case(5, 2048, torch.float32, torch.float32, 9, offset=3000.0)
    _, _, rstd = ops.layer_norm(x, g, b, EPS, stats=True)
    _, _, r, _ = _plain(x, g, b)
    # the centred values are off by n eps max|x| with n = d / 32 + 16, a second sweep forms the variance
    n = 2048 / 32 + 16
    bound = 2 * (2 * n * EPS32 * x.double().abs().amax(1) * r[:, 0]) + 4 * n * EPS32
    assert ((rstd.double() / r[:, 0] - 1).abs() <= bound).all()
    assert bound.max() < 0.2  # a variance formed as E[x^2] - mean^2 would be off by more than 1


def _check_grad(dx, dg, db, dy, x, mean, rstd, g, dtype):
    d, rows = x.shape[1], x.shape[0]
    D = lambda t: t.double()
    xh = (D(x) - D(mean)[:, None]) * D(rstd)[:, None]
    a = D(dy) * D(g)
    c1, c2 = a.mean(1, keepdim=True), (a * xh).mean(1, keepdim=True)
    want = D(rstd)[:, None] * (a - c1 - xh * c2)
    n = d / 32 + 16
    # xh has an error of 2 eps relative, and eps (|x| + |mean|) r from the subtraction
    xe = 4 * EPS32 * xh.abs() + EPS32 * (D(x).abs() + D(mean).abs()[:, None]) * D(rstd)[:, None]
    c1e = (n + 2) * EPS32 * a.abs().mean(1, keepdim=True)
    c2e = (n + 4) * EPS32 * (a * xh).abs().mean(1, keepdim=True) + (a.abs() * xe).mean(1, keepdim=True)
    tol = D(rstd)[:, None] * (c1e + xh.abs() * c2e + xe * c2.abs() + 8 * EPS32 * (a.abs() + c1.abs() + (xh * c2).abs()))
    tiny = 2.0 ** -25 if dtype == "float16" else 1e-38
    assert ((D(dx) - want).abs() <= tol + ULP[dtype] * (want.abs() + tol) + tiny).all()
    # a column's sum: at most `rows` terms one after another, then a join
    m = rows + 32
    u = ULP[str(g.dtype).replace("torch.", "")]
    wg, wb = (D(dy) * xh).sum(0), D(dy).sum(0)
    tg = (m + 4) * EPS32 * (D(dy) * xh).abs().sum(0) + (D(dy).abs() * xe).sum(0)
    tb = m * EPS32 * D(dy).abs().sum(0)
    assert ((D(dg) - wg).abs() <= tg + u * (wg.abs() + tg) + tiny).all()
    assert ((D(db) - wb).abs() <= tb + u * (wb.abs() + tb) + tiny).all()


@pytest.mark.parametrize("dtype,ptype", [("float32", "float32"), ("bfloat16", "bfloat16"),
                                         ("bfloat16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("d", WIDTHS)
def test_backward(d, dtype, ptype):
    torch, ops = _torch()
    for rows in (1, 3, 700):
        x, g, b, dy = _case(rows, d, getattr(torch, dtype), getattr(torch, ptype), 31 * d + rows)
        _, mean, rstd = ops.layer_norm(x, g, b, EPS, stats=True)
        dx, dg, db = ops.layer_norm_backward(dy, x, mean, rstd, g)
        assert dg.dtype == g.dtype and db.dtype == g.dtype and dx.dtype == x.dtype
        _check_grad(dx, dg, db, dy, x, mean, rstd, g, dtype)
        again = ops.layer_norm_backward(dy, x, mean, rstd, g)
        assert all(torch.equal(p, q) for p, q in zip((dx, dg, db), again))
        only, none_g, none_b = ops.layer_norm_backward(dy, x, mean, rstd, g, param_grads=False)
        assert torch.equal(only, dx) and none_g is None and none_b is None


def test_backward_without_gamma():
    torch, ops = _torch()
    x, g, _, dy = _case(50, 640, torch.bfloat16, torch.float32, 5)
    g = torch.ones_like(g)
    _, mean, rstd = ops.layer_norm(x, stats=True)
    a = ops.layer_norm_backward(dy, x, mean, rstd)
    b = ops.layer_norm_backward(dy, x, mean, rstd, g)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_gradient_against_differences():
    """The kernels' dx, dgamma and dbeta against central differences of the 64-bit formula: with a
    step h the difference's own error is of order h^2 (third derivative) plus 2^-53 / h."""
    torch, ops = _torch()
    rows, d, h = 2, 17, 1e-4
    x, g, b, dy = _case(rows, d, torch.float32, torch.float32, 11)
    _, mean, rstd = ops.layer_norm(x, g, b, EPS, stats=True)
    dx, dg, db = ops.layer_norm_backward(dy, x, mean, rstd, g)

    def f(x, g, b):
        return (_plain(x, g, b)[0] * dy.double()).sum()

    args = [x.double(), g.double(), b.double()]
    for k, grad in enumerate((dx, dg, db)):
        flat = grad.double().reshape(-1)
        for i in range(flat.numel()):
            up, dn = [[t.clone() for t in args] for _ in range(2)]
            up[k].view(-1)[i] += h
            dn[k].view(-1)[i] -= h
            num = (f(*up) - f(*dn)) / (2 * h)
            assert abs(num - flat[i]) <= 1e-6 + 1e-5 * grad.double().abs().max(), (k, i)


def test_autograd_and_in_place_gradient():
    torch, ops = _torch()
    x, g, b, dy = _case(40, 384, torch.float32, torch.float32, 13)
    x.requires_grad_(), g.requires_grad_(), b.requires_grad_()
    y = ops.layer_norm_autograd(x, g, b)
    y.backward(dy)
    with torch.no_grad():
        _, mean, rstd = ops.layer_norm(x, g, b, stats=True)
        dx, dg, db = ops.layer_norm_backward(dy, x, mean, rstd, g)
    assert torch.equal(x.grad, dx) and torch.equal(g.grad, dg) and torch.equal(b.grad, db)


@pytest.mark.parametrize("d", [64, 66, 100, 128, 129, 130, 771, 1024, 1030, 2048, 4098, 5000, 9998, 16384, 20001])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_fp8_form(d, dtype):
    """Scales to the layer norm's own tolerance; codes as those of the 64-bit y, save where y / scale
    lies within the error of a rounding boundary, and then the neighbouring code."""
    torch, ops = _torch()
    rows = 67
    x, g, b, _ = _case(rows, d, getattr(torch, dtype), torch.float32, d)
    q, mean, rstd = ops.layer_norm_fp8(x, g, b, EPS, stats=True)
    _, m2, r2 = ops.layer_norm(x, g, b, EPS, stats=True)
    assert torch.equal(mean, m2) and torch.equal(rstd, r2)
    assert q.codes.shape == (rows, d) and q.scales.shape == (rows, -(-d // 128)) and q.codes.stride(0) % 16 == 0
    want, _, r, xh = _plain(x, g, b)
    n = d / 32 + 16
    spread = 2 * n * EPS32 * x.double().abs().amax(1, keepdim=True) * r
    tol = _y_tol(x, g, b, r, xh, "float32") + (xh * g.double()).abs() * 2 * spread
    pad = -(-d // 128) * 128 - d
    amax = torch.nn.functional.pad(want.abs(), (0, pad)).view(rows, -1, 128).amax(2)
    tmax = torch.nn.functional.pad(tol, (0, pad)).view(rows, -1, 128).amax(2)
    assert ((q.scales.double() - amax / 448).abs() <= tmax / 448 + 2 * EPS32 * amax / 448 + 2.0 ** -126).all()
    s = q.scales.double().repeat_interleave(128, 1)[:, :d]
    got = q.codes.double()
    # half a step of the E4M3 grid at the value (2^-4 of it in the normal range, 2^-10 below; the
    # encoder keeps values under 2^-6 at most at 7 * 2^-9, a whole step)
    v = want / s
    half = torch.maximum(v.abs() * 2.0 ** -4, torch.full_like(v, 2.0 ** -10)) + (v.abs() < 2.0 ** -6) * 2.0 ** -10
    assert ((got - v).abs() <= half + tol / s + 8 * EPS32 * v.abs()).all()


def test_empty_and_refusals():
    torch, ops = _torch()
    from neuroflow_b200 import _nfx
    x, g, b, dy = _case(4, 64, torch.float32, torch.float32, 2)
    e = x[:0]
    y, mean, rstd = ops.layer_norm(e, g, b, stats=True)
    assert y.shape == (0, 64) and mean.shape == (0,)
    dx, dg, db = ops.layer_norm_backward(e, e, mean, rstd, g)
    assert dx.shape == (0, 64) and not dg.any() and not db.any()
    assert ops.layer_norm_fp8(e, g, b).codes.shape == (0, 64)
    _, mean, rstd = ops.layer_norm(x, stats=True)
    bad = [
        lambda: ops.layer_norm(x.cpu()),
        lambda: ops.layer_norm(x.double()),
        lambda: ops.layer_norm(x.t()),
        lambda: ops.layer_norm(x[:, :0]),
        lambda: ops.layer_norm(x, g[:-1]),
        lambda: ops.layer_norm(x, g, b.half()),
        lambda: ops.layer_norm(x, g, b, -1.0),
        lambda: ops.layer_norm(x, g, b, float("nan")),
        lambda: ops.layer_norm(x, out=torch.empty_like(x, dtype=torch.bfloat16)),
        lambda: ops.layer_norm(x[:1].expand(4, 64)),
        lambda: ops.layer_norm_backward(dy[:2], x, mean, rstd, g),
        lambda: ops.layer_norm_backward(dy.half(), x, mean, rstd, g),
        lambda: ops.layer_norm_backward(dy, x, mean[:2], rstd, g),
        lambda: ops.layer_norm_backward(dy, x, mean.double(), rstd, g),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(_nfx.NfxError) as ei:
            f()
        assert ei.value.code == 1, i
    # the C entries themselves: types, sizes, null pointers, a workspace that is too small
    L, p = _nfx.lib, x.data_ptr()
    ws = torch.empty(8, device="cuda")
    assert L.nfx_layer_norm(p, 9, 64, None, None, 0, 4, 64, EPS, p, 64, None, None, None) == 1
    assert L.nfx_layer_norm(p, 0, 64, None, None, 0, -1, 64, EPS, p, 64, None, None, None) == 1
    assert L.nfx_layer_norm(p, 0, 64, None, None, 0, 4, 0, EPS, p, 64, None, None, None) == 1
    assert L.nfx_layer_norm(p, 0, 63, None, None, 0, 4, 64, EPS, p, 64, None, None, None) == 1
    assert L.nfx_layer_norm(None, 0, 64, None, None, 0, 4, 64, EPS, p, 64, None, None, None) == 1
    assert L.nfx_layer_norm(p + 1, 0, 64, None, None, 0, 4, 64, EPS, p, 64, None, None, None) == 1
    assert L.nfx_layer_norm_backward(p, 64, p, 64, 0, mean.data_ptr(), rstd.data_ptr(), None, 0, 4, 64, p, 64,
                                     g.data_ptr(), b.data_ptr(), ws.data_ptr(), 32, None) == 1
    assert b"workspace" in L.nfx_last_error()
    assert _nfx.device_errors() == 0


def test_side_stream_and_long_offsets():
    """A call on another stream than the current one, and rows whose offsets pass 2^31 elements."""
    torch, ops = _torch()
    x, g, b, dy = _case(300, 1024, torch.bfloat16, torch.float32, 21)
    want = ops.layer_norm(x, g, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    y = ops.layer_norm(x, g, b, stream=s)
    y2 = ops.layer_norm(x, g, b, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(y, want) and torch.equal(y2, want)
    pitch = 1 << 29
    hold = torch.empty(4 * pitch + 1024, dtype=torch.bfloat16, device="cuda")
    wide = hold[:5 * pitch - pitch + 1024].as_strided((5, 1024), (pitch, 1))
    wide.copy_(x[:5])
    assert torch.equal(ops.layer_norm(wide, g, b), want[:5])
    qa, qb = ops.layer_norm_fp8(wide, g, b), ops.layer_norm_fp8(x[:5], g, b)
    assert torch.equal(qa.codes.float(), qb.codes.float()) and torch.equal(qa.scales, qb.scales)
    _, mean, rstd = ops.layer_norm(wide, g, b, stats=True)
    got, ref = ops.layer_norm_backward(dy[:5], wide, mean, rstd, g), ops.layer_norm_backward(dy[:5], x[:5], mean, rstd, g)
    assert all(torch.equal(p, q) for p, q in zip(got, ref))
