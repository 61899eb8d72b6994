"""GELU in the FP8 product's epilogue far from zero: 0 for very negative values, the value itself for
very large ones, and a NaN only in its own place.

The kernel forms gelu(z) as z (r b) with r = 1 / (a b) shared by two neighbours, a = 1 + exp(-2 u) of this
one and b of the other: the approximate division is off by 2 ulp at most, the two products by half an
ulp each, so with the other neighbour's b another 3 x 2^-23 is possible, and without it (a = 1) the value
itself is met to 3 x 2^-23, plus a rounding to the output's type."""
import pytest

pytestmark = pytest.mark.gpu

# few rows and one token, a split K, and enough rows and columns for pairs of CTAs
SHAPES = [(1, 300, 256), (5, 203, 2048), (130, 260, 300), (2600, 2200, 256)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_gelu_of_values_far_from_zero(m, n, k, dtype):
    import torch
    from neuroflow_b200 import ops
    gen = torch.Generator(device="cuda").manual_seed(m)
    a = ops.fp8_quantise(torch.randn(m, k, generator=gen, device="cuda"))
    w = ops.fp8_quantise(torch.randn(n, k, generator=gen, device="cuda") / k ** 0.5, tile=True)
    dt = getattr(torch, dtype)
    bias = 0.1 * torch.randn(n, generator=gen, device="cuda")
    plain = ops.fp8_gemm(a, w, bias=bias, act=1, out_dtype=dt)
    far = [-3e1, -1e4, -1e15, -1e18, -1e20, -1e38, -3e38]
    low, high, bad = [3 + 13 * i for i in range(len(far))], [100, 117, 190], [150, 169]
    for i, v in zip(low, far):
        bias[i] = v
    bias[high[0]], bias[high[1]], bias[high[2]] = 1e4, 1e20, 3e38
    for i in bad:
        bias[i] = float("nan")
    z = ops.fp8_gemm(a, w, bias=bias, out_dtype=torch.float32)
    got = ops.fp8_gemm(a, w, bias=bias, act=1, out_dtype=dt)
    # gelu(z) = z / (1 + exp(-2 u)); at z <= -16 that is below 1e-137
    assert (z[:, low] < -16).all() and (got[:, low] == 0).all()
    big, ulp = z[:, high].double(), {"float32": 0.0, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}[dtype]
    limit = torch.finfo(dt).max
    over = big > limit * (1 + 3 * 2.0 ** -23)
    assert (got[:, high][over] == float("inf")).all() if dtype == "float16" else not over.any()
    assert ((got[:, high].double() - big).abs()[~over] <= ((3 * 2.0 ** -23 + ulp) * big)[~over]).all()
    assert got[:, bad].isnan().all()
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[low + high + bad] = False
    assert torch.equal(got[:, rest].isnan(), torch.zeros_like(got[:, rest], dtype=torch.bool))
    diff = (got[:, rest].double() - plain[:, rest].double()).abs()
    assert (diff <= (6 * 2.0 ** -23 + 2 * ulp) * plain[:, rest].double().abs() + (2.0 ** -24 if dtype == "float16" else 0.0)).all()
