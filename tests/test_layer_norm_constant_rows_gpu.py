"""Layer norm of rows whose spread is small against their mean (neuroflow_b200.ops).

A variance formed as mean(c^2) - mean(c)^2 of nearly centred values c must not come out below zero.
"""
import pytest

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
EPS = 1e-5


def _torch():
    import torch
    from neuroflow_b200 import ops
    return torch, ops


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
