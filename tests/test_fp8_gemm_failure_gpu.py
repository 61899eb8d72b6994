"""The bounded waits of the FP8 product, without a GPU fault: with a budget of 1 ns
(nfx_debug_set_wait_budget_ns) the pipeline waits give up, the kernel records it in the device error
word, waits for its own copies and MMAs (with the normal limit), releases its tensor memory and returns;
with the normal budget the same context then computes the right result.  One case for each kernel: CTA
pairs, and the narrow one with and without a split K."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture
def budget():
    from neuroflow_b200 import _nfx
    f = _nfx.lib.nfx_debug_set_wait_budget_ns
    f.restype = None
    f.argtypes = [C.c_ulonglong]
    yield f
    f(0)


@pytest.mark.parametrize("m,n,k", [(2048, 2304, 4096), (16, 1024, 8192), (64, 20000, 1024)])
def test_waits_that_run_out_are_reported(budget, m, n, k):
    import torch
    from neuroflow_b200 import _nfx, ops
    g = torch.Generator(device="cuda").manual_seed(k)
    a = ops.fp8_quantise(torch.randn(m, k, generator=g, device="cuda"))
    w = ops.fp8_quantise(torch.randn(n, k, generator=g, device="cuda"), tile=True)
    want = ops.fp8_gemm(a, w)
    assert _nfx.device_errors() == 0
    budget(1)
    ops.fp8_gemm(a, w)
    flags = _nfx.device_errors()  # synchronises; the launch itself succeeded
    assert flags != 0 and flags & ~0x1F == 0, hex(flags)
    budget(0)
    for _ in range(2):
        assert torch.equal(ops.fp8_gemm(a, w), want)
        assert _nfx.device_errors() == 0
