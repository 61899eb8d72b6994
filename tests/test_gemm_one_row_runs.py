"""The 16-bit product of one row whose K is cut into runs: the runs' sums lie one behind the other in the
workspace, so with N no multiple of four all but the first start between 16-byte boundaries.  The row has to be
given by its column (A transposed); another one goes through the kernel for few rows.  Whole numbers, whose sums are
exact."""
import ctypes as C

import pytest

from test_gemm_dense_gpu import _ints, _torch

gpu = pytest.mark.gpu
# (N, K): runs on a device of 148 SMs
SHAPES = {(65, 16384): 8, (101, 8192): 4, (767, 16384): 2, (66, 16384): 8, (3, 65536): 13, (64, 16384): 8}


def _runs(n, k, sms):
    from neuroflow_b200 import _nfx
    f = _nfx.lib.nfx_debug_gemm_plan
    f.restype = None
    f.argtypes = [C.c_int64] * 3 + [C.c_int] * 4 + [C.POINTER(C.c_int)] * 4
    got = [C.c_int() for _ in range(4)]
    f(1, n, k, 1, 0, 1, sms, *got)
    return got[3].value


def test_one_row_is_cut_into_runs():
    for (n, k), runs in SHAPES.items():
        assert _runs(n, k, 148) == runs, (n, k)


@gpu
@pytest.mark.parametrize("n,k", list(SHAPES))
def test_one_row_of_a_long_k(n, k):
    torch, ops = _torch()
    from neuroflow_b200 import _nfx
    assert _runs(n, k, torch.cuda.get_device_properties(0).multi_processor_count) > 1
    gen = torch.Generator(device="cuda").manual_seed(n)
    for dt in (torch.bfloat16, torch.float16):
        for width in (8, 3):  # a column of rows that start on 16-byte boundaries, or do not
            a = _ints(gen, k, width, dt)[:, :1].t()
            b = _ints(gen, n, k, dt)
            want = a.double() @ b.double().t()
            bias, res = torch.arange(n, device="cuda").float() - 5, torch.ones(1, n, device="cuda").to(dt)
            for bb in (b, b.t().contiguous().t()):
                assert torch.equal(ops.gemm(a, bb, out_dtype=torch.float32).double(), want)
                got, z = ops.gemm(a, bb, bias=bias, act=2, residual=res, preact=True)
                assert torch.equal(z, (want + bias.double()).to(dt))
                assert torch.equal(got, ((want + bias.double()).clamp_min(0) + 1).to(dt))
    assert _nfx.device_errors() == 0


@gpu
@pytest.mark.parametrize("tokens,k", [(16384, 65), (8192, 101), (16385, 767), (20000, 64)])
def test_gradients_of_a_layer_with_one_output(tokens, k):
    """dW of such a layer is a product of one row, as long as there are tokens."""
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    x, w, dy = _ints(gen, tokens, k, torch.float16, 1), _ints(gen, 1, k, torch.float16), _ints(gen, tokens, 1, torch.float16, 1)
    x.requires_grad_(), w.requires_grad_()
    y = ops.linear(x, w)
    X, W, D = x.detach().double(), w.detach().double(), dy.double()
    assert torch.equal(y.detach(), (X @ W.t()).half())
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert torch.equal(dw, (D.t() @ X).half()) and torch.equal(dx, (D @ W).half())
