"""Refusals of the RMS norm, 16-bit product, activation gradient and clipping entries that need no GPU:
arguments are checked before anything is launched, with the reason in nfx_last_error()."""
import ctypes as C

import pytest

from neuroflow_b200 import _nfx

L = _nfx.lib
P = 1 << 12  # an aligned address that is never read


def _bad(rc, word):
    assert rc == 1, rc
    assert word in L.nfx_last_error().decode(), L.nfx_last_error()


def test_rms_norm_refusals():
    f = lambda x=P, xt=1, ldx=64, res=P, ht=1, ldr=64, pt=0, rows=4, d=64, eps=1e-5, y=P, ldy=64, s=P, lds=64: L.nfx_rms_norm(
        x, xt, ldx, res, ht, ldr, None, pt, rows, d, eps, y, ldy, s, lds, None, None)
    _bad(f(xt=3), "type")
    _bad(f(pt=-1), "type")
    _bad(f(ht=7), "type")
    _bad(f(ht=2), "residual must have")
    _bad(f(rows=-1), "rows")
    _bad(f(d=0), "d >= 1")
    _bad(f(d=(1 << 31) - 256, ldx=1 << 32, ldy=1 << 32), "2^31 - 256")
    for k in ("ldx", "ldr", "ldy", "lds"):
        _bad(f(**{k: 63}), "stride")
    _bad(f(x=None), "null")
    _bad(f(y=None), "null")
    _bad(f(res=None), "with a residual only")
    for k in ("x", "res", "y", "s"):
        _bad(f(**{k: P + 1}), "aligned")
    _bad(f(eps=float("nan")), "eps")
    _bad(f(eps=-1.0), "eps")
    assert f(rows=0, x=None, y=None, res=None, s=None) == 0
    q = lambda codes=P, scales=P, ld=64: L.nfx_rms_norm_fp8(P, 1, 64, None, 0, 0, None, 0, 4, 64, 1e-5, codes, ld, scales, 1, 4, None, 0,
                                                            None, None)
    _bad(q(codes=None), "null")
    _bad(q(scales=None), "null")
    _bad(q(scales=P + 2), "aligned")
    _bad(q(ld=63), "stride")


def test_rms_norm_backward_refusals():
    f = lambda dy=P, yt=1, h=P, ht=1, r=P, ds=None, ldd=64, dx=P, lddx=64, dr=None, ldr=64, dg=None, ws=None, n=0, rows=4: \
        L.nfx_rms_norm_backward(dy, yt, 64, h, ht, 64, r, None, 0, ds, ldd, rows, 64, dx, lddx, dr, ldr, dg, ws, n, None)
    _bad(f(dy=None), "null")
    _bad(f(h=None), "null")
    _bad(f(r=None), "null")
    _bad(f(r=P + 2), "aligned")
    _bad(f(ht=2), "residual must have")
    _bad(f(lddx=10), "stride")
    _bad(f(ds=P, ldd=10), "stride")
    _bad(f(dr=P, ldr=10), "stride")
    _bad(f(ds=P + 1), "aligned")
    _bad(f(dg=P), "workspace")
    _bad(f(dg=P, ws=P, n=7), "workspace")
    _bad(f(dg=P, ws=P + 8, n=1 << 20), "16-byte")
    assert L.nfx_rms_norm_backward_workspace(0, 64) == 0 and L.nfx_rms_norm_backward_workspace(4, 64) >= 64 * 4


def test_gemm_refusals():
    f = lambda a=P, lda=256, at=0, b=P, ldb=256, bt=0, t=1, m=8, n=64, k=256, bias=None, biast=0, act=0, r=None, ldr=64, c=P, ct=1, ldc=64, \
        z=None, ldz=64, ws=None, size=0: L.nfx_gemm(a, lda, at, b, ldb, bt, t, m, n, k, bias, biast, act, r, ldr, c, ct, ldc, z, ldz, ws, size, None)
    _bad(f(m=-1), ">= 0")
    _bad(f(n=(1 << 31) - 256), "2^31 - 256")
    _bad(f(t=0), "ab_type")
    _bad(f(t=3), "ab_type")
    _bad(f(ct=2), "c_type")
    _bad(f(ct=5), "type")
    _bad(f(biast=5), "type")
    _bad(f(act=3), "act")
    _bad(f(at=2), "a_trans")
    _bad(f(bt=-1), "a_trans")
    _bad(f(a=None), "null")
    _bad(f(b=None), "null")
    _bad(f(c=None), "null")
    _bad(f(lda=255), "stride")
    _bad(f(at=1, lda=7), "stride")
    _bad(f(bt=1, ldb=63), "stride")
    _bad(f(ldc=63), "stride")
    _bad(f(r=P, ldr=63), "stride")
    _bad(f(z=P, ldz=63), "stride")
    for k in ("a", "b", "c", "r", "z"):
        _bad(f(**{k: P + 1}), "aligned")
    _bad(f(bias=P + 2), "aligned")
    _bad(f(m=(1 << 31) - 300, n=(1 << 31) - 300, k=8, ldc=1 << 31), "too many")
    assert f(m=0, a=None, c=None) == 0 and f(n=0) == 0


def test_gemm_workspace():
    w = lambda a=P, lda=256, at=0, b=P, ldb=256, bt=0, m=8, n=64, k=256: L.nfx_gemm_workspace(a, lda, at, b, ldb, bt, m, n, k)
    assert w() == 0 and w(m=0, lda=3) == 0 and w(k=0) == 0


def test_act_backward_refusals():
    f = lambda dy=P, ldy=64, z=P, ldz=64, t=1, act=1, rows=4, cols=64, dz=P, lddz=64, db=None, bt=0, ws=None, n=0: L.nfx_act_backward(
        dy, ldy, z, ldz, t, act, rows, cols, dz, lddz, db, bt, ws, n, None)
    _bad(f(t=3), "type")
    _bad(f(bt=4), "type")
    _bad(f(act=-1), "act")
    _bad(f(rows=-1), ">= 0")
    _bad(f(cols=1 << 31), "2^31")
    _bad(f(dy=None), "null")
    _bad(f(z=None), "null")
    for k in ("ldy", "ldz", "lddz"):
        _bad(f(**{k: 63}), "stride")
    for k in ("dy", "z", "dz"):
        _bad(f(**{k: P + 1}), "aligned")
    _bad(f(db=P), "workspace")
    assert f(rows=0, dy=None, z=None) == 0


def _list(ptrs, counts, types, out=None, out_types=None):
    n = len(ptrs)
    arr = lambda t, v: None if v is None else (t * max(n, 1))(*v)
    return arr(C.c_void_p, ptrs), arr(C.c_int64, counts), arr(C.c_int, types), arr(C.c_void_p, out), arr(C.c_int, out_types), n


def test_clip_refusals():
    def f(ptrs=(P, P * 2), counts=(4, 4), types=(0, 1), out=None, ot=None, mx=1.0, eps=1e-6, norm=P, ws=P, size=1 << 20, tensors=None):
        p, c, t, o, q, n = _list(ptrs, counts, types, out, ot)
        return L.nfx_clip_grad_norm(p, c, t, o, q, n if tensors is None else tensors, mx, eps, norm, ws, size, None)
    _bad(f(types=(0, 3)), "type")
    _bad(f(counts=(4, -1)), "negative")
    _bad(f(ptrs=(P, None)), "null")
    _bad(f(ptrs=(P, P + 1)), "aligned")
    _bad(f(out=(P, P + 1), ot=(0, 1)), "aligned")
    _bad(f(out=(P, None), ot=(0, 1)), "null")
    _bad(f(out=(P, P), ot=(0, 9)), "type")
    _bad(f(out=(P, P)), "null")
    _bad(f(tensors=-1), "tensors")
    _bad(f(mx=-1.0), "max_norm")
    _bad(f(mx=float("nan")), "max_norm")
    _bad(f(eps=float("nan")), "eps")
    _bad(f(eps=float("inf")), "eps")
    _bad(f(norm=None), "null")
    _bad(f(norm=P + 2), "aligned")
    _bad(f(ws=None), "workspace")
    _bad(f(size=8), "workspace")
    _bad(f(ws=P + 8), "16-byte")
    p, c, t, _, _, n = _list((P,), (-4,), (0,))
    _bad(L.nfx_grad_norm(p, c, t, n, P, P, 1 << 20, None), "negative")
    assert L.nfx_grad_norm_workspace(5000) > L.nfx_grad_norm_workspace(1) > 0 and L.nfx_grad_norm_workspace(-1) == 0


def test_front_end_refuses_cpu_tensors():
    import torch
    from neuroflow_b200 import ops
    x, h = torch.zeros(4, 64), torch.zeros(4, 64, dtype=torch.bfloat16)
    for f in (lambda: ops.rms_norm(x), lambda: ops.rms_norm_fp8(x), lambda: ops.rms_norm_backward(x, x, x[:, 0]), lambda: ops.rms_norm_autograd(x),
              lambda: ops.gemm(h, h), lambda: ops.linear(h, h), lambda: ops.act_backward(x, x, 1), lambda: ops.grad_norm([x]),
              lambda: ops.clip_grad_norm([x], 1.0), lambda: ops.clip_grad_norm([], 1.0), lambda: ops.grad_norm([])):
        with pytest.raises(_nfx.NfxError) as ei:
            f()
        assert ei.value.code == 1
    for f in (lambda: ops.grad_norm([None]), lambda: ops.clip_grad_norm([x, 3], 1.0), lambda: ops.clip_grad_norm([x], 1.0, out=["x"])):
        with pytest.raises(TypeError, match="must be tensors"):
            f()
