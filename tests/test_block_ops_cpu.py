"""Refusals of the layer norm, quantiser and product entries that need no GPU: arguments are checked
before anything is launched, with the reason in nfx_last_error()."""
import ctypes as C

from neuroflow_b200 import _nfx

L = _nfx.lib
P = 1 << 12  # an aligned address that is never read


def _bad(rc, word):
    assert rc == 1, rc
    assert word in L.nfx_last_error().decode()


def test_layer_norm_refusals():
    f = lambda x=P, xt=0, ldx=64, pt=0, rows=4, d=64, eps=1e-5, y=P, ldy=64: L.nfx_layer_norm(
        x, xt, ldx, None, None, pt, rows, d, eps, y, ldy, None, None, None)
    _bad(f(xt=3), "x_type")
    _bad(f(pt=-1), "param_type")
    _bad(f(rows=-1), "rows")
    _bad(f(d=0), "d >= 1")
    _bad(f(d=1 << 31, ldx=1 << 32, ldy=1 << 32), "2^31")
    _bad(f(ldx=63), "stride")
    _bad(f(ldy=63), "stride")
    _bad(f(x=None), "null")
    _bad(f(y=None), "null")
    _bad(f(x=P + 2), "aligned")
    _bad(f(y=P + 1), "aligned")
    _bad(f(eps=float("nan")), "eps")
    assert f(rows=0, x=None, y=None) == 0
    q = lambda codes=P, scales=P, ld=64: L.nfx_layer_norm_fp8(
        P, 1, 64, None, None, 0, 4, 64, 1e-5, codes, ld, scales, 1, 4, None, None, None)
    _bad(q(codes=None), "null")
    _bad(q(scales=None), "null")
    _bad(q(scales=P + 2), "aligned")
    _bad(q(ld=63), "stride")


def test_layer_norm_backward_refusals():
    f = lambda dy=P, mean=P, dx=P, dg=None, ws=None, n=0, lddx=64: L.nfx_layer_norm_backward(
        dy, 64, P, 64, 0, mean, P, None, 0, 4, 64, dx, lddx, dg, None, ws, n, None)
    _bad(f(dy=None), "null")
    _bad(f(mean=None), "null")
    _bad(f(dx=None), "null")
    _bad(f(lddx=10), "stride")
    _bad(f(dg=P), "workspace")
    _bad(f(dg=P, ws=P, n=7), "workspace")
    assert L.nfx_layer_norm_backward_workspace(0, 64) == 0
    assert L.nfx_layer_norm_backward_workspace(4, 64) >= 2 * 64 * 4


def test_quantise_refusals():
    f = lambda x=P, xt=1, ld=130, rows=4, cols=130, tile=0, codes=P, ldc=144, scales=P, ct=None, ldt=16, st=None, sums=None, sumt=0, ws=None, n=0: \
        L.nfx_fp8_quantise(x, xt, ld, rows, cols, tile, codes, ldc, scales, 1, 4, ct, ldt, st, 1, 130, sums, sumt, ws, n, None)
    _bad(f(xt=9), "x_type")
    _bad(f(sumt=4), "sums_type")
    _bad(f(rows=-1), "rows")
    _bad(f(cols=1 << 31), "2^31")
    _bad(f(tile=2), "tile")
    _bad(f(tile=1, sums=P), "column sums")
    _bad(f(x=None), "null")
    _bad(f(codes=None), "null")
    _bad(f(ct=P), "null")
    _bad(f(ld=129), "stride")
    _bad(f(ct=P, st=P, ldt=3), "stride")
    _bad(f(x=P + 1), "aligned")
    _bad(f(sums=P), "workspace")
    _bad(f(sums=P, ws=P, n=100), "workspace")
    assert f(rows=0, x=None, codes=None, scales=None) == 0
    assert L.nfx_fp8_quantise_workspace(129, 10) == 2 * 10 * 4


def test_gemm_refusals():
    f = lambda a=P, lda=256, b=P, ldb=256, sa=P, m=8, n=64, k=256, bt=0, act=0, c=P, ct=0, ldc=64, at=0: L.nfx_fp8_gemm(
        a, lda, sa, 1, 8, at, b, ldb, P, 1, 1, 1, m, n, k, None, bt, act, c, ct, ldc, None)
    _bad(f(m=-1), ">= 0")
    _bad(f(n=1 << 31), "2^31")
    _bad(f(act=3), "act")
    _bad(f(ct=5), "type")
    _bad(f(bt=5), "type")
    _bad(f(at=2), "a_tile")
    _bad(f(a=None), "null")
    _bad(f(c=None), "null")
    _bad(f(sa=None), "null")
    _bad(f(ldc=63), "ldc")
    _bad(f(lda=255), "stride")
    _bad(f(lda=264), "16-byte")
    _bad(f(b=P + 8), "16-byte")
    _bad(f(c=P + 1), "aligned")
    assert f(m=0, a=None, c=None) == 0 and f(n=0) == 0


def test_front_end_refuses_cpu_tensors():
    import pytest
    import torch
    from neuroflow_b200 import ops
    x = torch.zeros(4, 64)
    for f in (lambda: ops.layer_norm(x), lambda: ops.layer_norm_fp8(x), lambda: ops.fp8_quantise(x),
              lambda: ops.fp8_linear(x, x), lambda: ops.layer_norm_backward(x, x, x[:, 0], x[:, 0]),
              lambda: ops.fp8_gemm(ops.Fp8Blocks(x, x), ops.Fp8Blocks(x, x))):
        with pytest.raises(_nfx.NfxError) as ei:
            f()
        assert ei.value.code == 1
    assert isinstance(_nfx.NfxError(1, "x"), RuntimeError) and C.sizeof(C.c_int64) == 8


def test_layer_norm_widths_that_a_column_index_cannot_step_over():
    """The kernels for any width step through a row by 256 columns with 32-bit indices: the widest row
    leaves room for one step beyond its end."""
    for d in ((1 << 31) - 256, (1 << 31) - 1):
        _bad(L.nfx_layer_norm(P, 1, d, None, None, 0, 1, d, 1e-5, P, d, None, None, None), "2^31 - 256")
        _bad(L.nfx_layer_norm_fp8(P, 1, d, None, None, 0, 1, d, 1e-5, P, d, P, 1, 1, None, None, None), "2^31 - 256")
        _bad(L.nfx_layer_norm_backward(P, d, P, d, 1, P, P, None, 0, 1, d, P, d, None, None, None, 0, None), "2^31 - 256")
    d = (1 << 31) - 257  # (no rows: nothing is launched)
    assert L.nfx_layer_norm(None, 1, d, None, None, 0, 0, d, 1e-5, None, d, None, None, None) == 0
