"""The mean of 16-bit rows whose sums are exact in fp32 (multiples of 2^-10 that add up to less than 2^14 in
magnitude): the quotient is the only rounding, and nothing may be added to it."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("d", [100, 771, 1000, 2048, 3001, 4096, 5000, 8192])
def test_mean_is_the_rounded_quotient(d, dtype):
    import torch
    from neuroflow_b200 import ops
    gen = torch.Generator(device="cuda").manual_seed(d)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x = ((0.5 * rnd(400, d) * torch.exp(0.7 * rnd(1, d)) + 0.25) * 1024).round() / 1024
    x = x.to(getattr(torch, dtype))
    assert x.double().abs().sum(1).max() < 2 ** 14 and torch.equal((x.double() * 1024).round(), x.double() * 1024)
    want = x.double().mean(1).float()  # the sum is exact in 64 bits, so this is off by a double rounding at most
    for form in (ops.layer_norm, ops.layer_norm_fp8):
        _, mean, rstd = form(x, stats=True)
        near = (mean.double() - x.double().mean(1)).abs() <= 2.0 ** -24 * (1 + 2.0 ** -20) * 2.0 ** torch.floor(torch.log2(want.abs().double())) + 1e-30
        assert near.all()
        if d & (d - 1) == 0:
            assert torch.equal(mean, want)
        v = x.double().var(1, correction=0)
        assert ((rstd.double() * (v + 1e-5).sqrt() - 1).abs() <= (d / 32 + 20) * 2.0 ** -24).all()
