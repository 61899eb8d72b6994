"""What the 16-bit product loses of a long sum of numbers of one sign, on every path.

A tensor core cuts off where an addition would round: at most 2^-23 of the running sum for each of the 16 products of a
step and for the sum before them, 17 * 2^-23 a step, where the running sum is half of the final one on the average.
Pieces of P terms are summed that way: a result is low by at most P / 16 * 17 * 2^-24 of itself, 3.3e-5 for the 512 terms
of fp32 results and 2.6e-4 for the 4,096 of 16-bit ones, whatever K is.  Pieces are joined in fp32, at most 2^-24 each; a
16-bit result's own rounding is up to half a step and nothing on the average (under 1e-5 over 2,000 results).
With all of K in one piece the mean of each shape is 1.2 times its bound or more."""
import pytest

from test_gemm_dense_gpu import _torch
from test_gemm_dense_paths import B200_SMS, _plan

gpu = pytest.mark.gpu
# (columns, split, deep): (M, N, K, A transposed, B transposed), results of 16 bits
HALF = [((0, 1, 0), (2304, 2304, 65536, 0, 0)), ((0, 1, 0), (2304, 2304, 65536, 1, 1)), ((0, 2, 0), (512, 3000, 131072, 0, 0)),
        ((0, 4, 0), (700, 700, 262144, 0, 0)), ((64, 8, 1), (64, 1024, 524288, 0, 0)), ((-1, 1, 0), (1, 2384, 524288, 0, 0)),
        ((-1, 1, 0), (12, 4800, 524288, 0, 0)), ((-1, 1, 0), (5, 9600, 524288, 0, 1))]
# fp32 results of the kernel for few rows, aligned and not
FULL = [((-1, 1, 0), (1, 2384, 131072, 0, 0)), ((-1, 1, 0), (16, 4800, 131072, 0, 0)), ((-1, 1, 0), (3, 9600, 131072, 0, 1)),
        ((-1, 1, 0), (2, 2384, 131073, 0, 0)), ((-1, 1, 0), (13, 4801, 131073, 0, 0)), ((-1, 1, 0), (30, 4801, 131073, 0, 0)),
        ((-1, 1, 0), (7, 9601, 131073, 0, 1))]


def test_paths_of_the_shapes():
    for path, (m, n, k, a_t, b_t) in HALF + FULL:
        aligned = int(k % 8 == 0 and (not b_t or n % 8 == 0))
        assert _plan(m, n, k, a_t, b_t, aligned, B200_SMS) == path, (m, n, k)


def _offsets(m, n, k, a_t, b_t, dtype, out):
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(k)

    def held(rows, cols, t, size):
        x = torch.empty(cols, rows, device="cuda", dtype=dtype).t() if t else torch.empty(rows, cols, device="cuda", dtype=dtype)
        for i in range(0, cols, 1 << 14):
            x[:, i:i + (1 << 14)] = size * torch.rand(rows, min(cols - i, 1 << 14), generator=gen, device="cuda")
        return x

    a, b = held(m, k, a_t, 1.0), held(n, k, b_t, 0.125)
    want = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    for i in range(0, k, 1 << 14):
        want += a[:, i:i + (1 << 14)].double() @ b[:, i:i + (1 << 14)].double().t()
    return ops.gemm(a, b, out_dtype=out).double() / want - 1


@gpu
@pytest.mark.parametrize("path,shape", HALF)
def test_results_of_16_bits(path, shape):
    torch, _ = _torch()
    off = _offsets(*shape, torch.float16, torch.float16)
    low = 4096 / 16 * 17 * 2.0 ** -24
    assert off.mean().abs() <= low + 1e-5, float(off.mean())
    assert off.abs().max() <= (1 + low) * (1 + 2.0 ** -11) - 1 + 64 * 2.0 ** -24, float(off.abs().max())


@gpu
@pytest.mark.parametrize("path,shape", FULL)
def test_fp32_results_of_few_rows(path, shape):
    torch, _ = _torch()
    m, n, k = shape[:3]
    off = _offsets(*shape, torch.float16, torch.float32)
    joins = k // 8 // 512 + 8 + 1
    assert off.abs().max() <= 512 / 16 * 17 * 2.0 ** -24 + joins * 2.0 ** -24, float(off.abs().max())
