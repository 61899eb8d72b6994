"""Layer norm of rows whose spread is small against their mean (neuroflow_b200.ops).

A variance formed as mean(c^2) - mean(c)^2 of nearly centred values c must not come out below zero,
and the rounding error of the mean, the same in every element of a constant row, must not be taken for
a spread.

Tolerances, for a row of d elements with mean mu, variance v and r = 1 / sqrt(v + EPS); eps = 2^-24.  A
sum of terms t is off by at most n eps sum |t| with n = d / 32 + 16 (threads add at most d / 32 elements
one after another and join in a tree).
  E0 = (n + 2) eps mean|x|                              the first mean's error
  C = mean|x - mu| + E0                                 mean size of the centred values
  rest (their mean, which is minus that error)          off by (n + 4) eps C
  dv = (n + 6) eps (v + E0^2) + 2 E0 (n + 4) eps C      the variance's error
  rel                                                   1/std's relative error: 1.2 times the first order,
       dv / (2 (v + EPS)) + 4 eps, or what 1 / sqrt(v +- dv + EPS) is off by (the variance not below zero)
       plus 5 eps where that is less
  y: |g| (r ((n + 6) eps C + 2 eps |x - mu| + 2 eps E0) + |xh| rel) + 4 eps (|g xh| + |b|), and eps |y|
"""
import pytest

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
EPS = 1e-5


def _torch():
    import torch
    from neuroflow_b200 import ops
    return torch, ops


def _bounds(x, g, b):
    import torch
    x, g, b = x.double(), g.double(), b.double()
    n = x.shape[1] / 32 + 16
    mu = x.mean(1, keepdim=True)
    c = x - mu
    v = c.square().mean(1, keepdim=True)
    r = (v + EPS) ** -0.5
    xh = c * r
    e0 = (n + 2) * E * x.abs().mean(1, keepdim=True)
    size = c.abs().mean(1, keepdim=True) + e0
    dv = (n + 6) * E * (v + e0 * e0) + 2 * e0 * (n + 4) * E * size
    up, low = dv / (v + EPS), torch.minimum(dv, v) / (v + EPS)
    far = torch.maximum(1 - (1 + up) ** -0.5, (1 - low) ** -0.5 - 1) + 5 * E
    rel = torch.minimum(1.2 * (up / 2 + 4 * E), far)
    y = xh * g + b
    ty = g.abs() * (r * ((n + 6) * E * size + 2 * E * c.abs() + 2 * E * e0) + xh.abs() * rel)
    ty = ty + 4 * E * ((g * xh).abs() + b.abs()) + E * y.abs()
    return y, ty, mu[:, 0], ((n + 4) * E * size + E * mu.abs())[:, 0], r[:, 0], rel[:, 0]


@pytest.mark.parametrize("d", [100, 1001, 1024, 4100, 5001, 8190, 16380, 20001])
def test_constant_rows_of_large_numbers_are_finite(d):
    """Full-mantissa constants around 1e9, whose sums are rounded: the variance is not negative, so 1/std is
    at most that of a zero variance and nothing is NaN."""
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(d)
    x = ((1 + torch.rand(150, 1, generator=gen, device="cuda")) * 1e9).expand(150, d).contiguous()
    x[0] = 1897923072.0
    y, mean, rstd = ops.layer_norm(x, stats=True)
    assert y.isfinite().all() and rstd.isfinite().all()
    assert (rstd > 0).all() and (rstd.double() <= EPS ** -0.5 * (1 + 4 * E)).all()
    assert ops.layer_norm_fp8(x).dequantise().isfinite().all()
    dx, dg, db = ops.layer_norm_backward(x * 1e-9, x, mean, rstd)
    assert dx.isfinite().all() and dg.isfinite().all() and db.isfinite().all()


def _rows(d):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(d)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x = torch.empty(8, d, device="cuda")
    for i, (at, spread) in enumerate([(1000.1, 0.0), (3000.3, 0.0), (1000.1, 1e-3), (-777.7, 1e-3), (50.3, 1e-2),
                                      (1000.1, 1.0), (0.0, 1.0), (0.1, 0.0)]):
        x[i] = at + spread * rnd(d)
    return x, 1 + 0.2 * rnd(d), 0.3 * rnd(d)


@pytest.mark.parametrize("d", [771, 2048, 4098, 16384, 16385, 20001, 40000])
def test_mean_far_above_the_spread(d):
    """Constant and nearly constant rows at every width, those that the registers hold and wider ones."""
    torch, ops = _torch()
    x, g, b = _rows(d)
    want, ty, mu, tm, r, rel = _bounds(x, g, b)
    y, mean, rstd = ops.layer_norm(x, g, b, EPS, stats=True)
    assert ((mean.double() - mu).abs() <= tm).all()
    assert ((rstd.double() / r - 1).abs() <= rel).all()
    assert ((y.double() - want).abs() <= ty).all()
    q = ops.layer_norm_fp8(x, g, b, EPS)
    s = q.scales.double().repeat_interleave(128, 1)[:, :d]
    # a step of the E4M3 grid: 2^-4 of the value, 2^-9 below the normal numbers
    assert ((q.dequantise().double() - want).abs() <= want.abs() / 16 + s * 2.0 ** -9 + 2 * ty).all()
