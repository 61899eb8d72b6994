"""Operators of one pre-norm FP8 linear layer on CUDA tensors: layer norm, the FP8 E4M3 block
quantiser and the FP8 block-scaled product, forward and backward.

    from neuroflow_b200 import ops
    y, mean, rstd = ops.layer_norm(x, gamma, beta, stats=True)
    dx, dgamma, dbeta = ops.layer_norm_backward(dy, x, mean, rstd, gamma)
    w8 = ops.fp8_quantise(w, tile=True)                  # once per weight
    x8 = ops.layer_norm_fp8(x, gamma, beta)              # layer norm straight into FP8
    y = ops.fp8_gemm(x8, w8, bias=b, act=1)              # act(x8 w8^T + b)
    y = ops.fp8_linear(x, w, b); y.backward(dy)          # the same linear layer under autograd

Every call runs the kernels of libnfx.so (the C-ABI of include/nfx.h) on the current torch
stream of the tensors' device, or on `stream` (a torch.cuda.Stream or raw handle), without
synchronising; outputs are allocated for that stream.  There is no CPU fallback.  Refused
arguments raise NfxError with code 1 (InvalidArg).  torch.float32, bfloat16 and float16 are
accepted where a tensor is not FP8; the last dimension has to be contiguous.
"""
from __future__ import annotations

import contextlib
from typing import NamedTuple

import torch

from . import _nfx

_lib = _nfx.lib
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
E4M3 = torch.float8_e4m3fn
GROUP = 128


class Fp8Blocks(NamedTuple):
    """A matrix in FP8 E4M3 with one fp32 scale per block of 128 along its rows.

    codes   (rows, cols) float8_e4m3fn, last dimension contiguous; the product needs rows
            that start on 16-byte boundaries (the quantiser lays them out so)
    scales  fp32, any strides: (rows, ceil(cols / 128)), or (ceil(rows / 128),
            ceil(cols / 128)) when `tile`
    tile    whether a scale covers 128 x 128 codes"""
    codes: torch.Tensor
    scales: torch.Tensor
    tile: bool = False

    def dequantise(self) -> torch.Tensor:
        """The fp32 matrix that the codes and scales stand for (elementary torch, for checks)."""
        r, c = self.codes.shape
        s = self.scales.repeat_interleave(GROUP, 1)[:, :c]
        if self.tile:
            s = s.repeat_interleave(GROUP, 0)[:r]
        return self.codes.float() * s


def _refuse(fn, what):
    raise _nfx.NfxError(1, f"{fn}: {what}")


def _up(a, b):
    return -(-a // b) * b


def _type(fn, name, t):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _refuse(fn, f"{name} must be a CUDA tensor")
    k = _TYPES.get(t.dtype)
    if k is None:
        _refuse(fn, f"{name} must be float32, bfloat16 or float16, not {t.dtype}")
    return k


def _same_device(fn, x, **others):
    for name, t in others.items():
        if t is not None and t.device != x.device:
            _refuse(fn, f"{name} is on {t.device}, not on {x.device}")


def _rows(fn, name, t, d=None):
    """t as (rows, d) with a row stride, without a copy."""
    if t.dim() < 1:
        _refuse(fn, f"{name} needs at least one dimension")
    if d is not None and t.shape[-1] != d:
        _refuse(fn, f"{name} has {t.shape[-1]} columns, not {d}")
    if t.dim() != 2:
        try:
            t = t.view(t.numel() // t.shape[-1] if t.shape[-1] else 0, t.shape[-1])
        except RuntimeError:
            _refuse(fn, f"the rows of {name} are not evenly strided: pass a contiguous tensor")
    if t.shape[1] > 1 and t.stride(1) != 1:
        _refuse(fn, f"the last dimension of {name} must be contiguous")
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        _refuse(fn, f"the rows of {name} overlap")
    return t


def _vector(fn, name, t, n, dtype=None):
    if t is None:
        return None
    _type(fn, name, t)
    if t.shape != (n,) or (n > 1 and t.stride(0) != 1):
        _refuse(fn, f"{name} must be a contiguous vector of {n}")
    if dtype is not None and t.dtype != dtype:
        _refuse(fn, f"{name} must be {dtype}, not {t.dtype}")
    return t


def _p(t):
    return None if t is None else t.data_ptr()


def _elsewhere(t, stream):
    """Whether a call on `t` needs another device or stream made current first (see _on)."""
    return stream is not None or t.device.index != torch.cuda.current_device()


@contextlib.contextmanager
def _on(t, stream):
    """The device of `t` and the stream of a call made current, so that what the call allocates
    belongs to that stream."""
    with torch.cuda.device(t.device):
        if stream is None:
            yield
            return
        if not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(int(stream), device=t.device)
        with torch.cuda.stream(stream):
            yield


def _stream(t):
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def _codes(rows, cols, device):
    """An empty code matrix whose rows start on 16-byte boundaries."""
    pitch = _up(cols, 16) or 16
    c = torch.empty((rows, pitch), dtype=E4M3, device=device)
    return c if pitch == cols else c[:, :cols]


def _scales(rows, cols, device):
    """Empty scales (rows, ceil(cols / 128)) with the block index outermost, the order in which
    the product reads them."""
    return torch.empty_strided((rows, -(-cols // GROUP)), (1, rows), dtype=torch.float32, device=device)


def _row_stats(x, rows):
    """Two empty fp32 vectors (mean, rstd), one element for each row of x."""
    return x.new_empty((2, rows) if x.dim() == 2 else (2, *x.shape[:-1]), dtype=torch.float32).unbind(0)


def _norm_args(fn, x, gamma, beta):
    xt = _type(fn, "x", x)
    x2 = _rows(fn, "x", x)
    d = x2.shape[1]
    if d < 1:
        _refuse(fn, "the last dimension is empty")
    g = _vector(fn, "gamma", gamma, d)
    b = _vector(fn, "beta", beta, d, None if gamma is None else gamma.dtype)
    _same_device(fn, x, gamma=g, beta=b)
    p = g if g is not None else b
    return x2, xt, g, b, (0 if p is None else _TYPES[p.dtype])


def layer_norm(x, gamma=None, beta=None, eps=1e-5, out=None, stats=False, stream=None):
    """Layer norm over the last dimension of x (..., d); gamma and beta (d,), None for ones and
    zeros.  y in x's type (in `out` if given); with `stats` also the fp32 mean and 1/std of each
    row, which layer_norm_backward takes: (y, mean, rstd)."""
    fn = "layer_norm"
    x2, xt, g, b, pt = _norm_args(fn, x, gamma, beta)
    if _elsewhere(x, stream):
        with _on(x, stream):
            return layer_norm(x, gamma, beta, eps, out, stats)
    rows, d = x2.shape
    if out is None:
        y = y2 = torch.empty_like(x, memory_format=torch.contiguous_format)
        ldy = d
    else:
        y = out
        if y.shape != x.shape or y.dtype != x.dtype or y.device != x.device:
            _refuse(fn, "out must have x's shape, type and device")
        y2 = _rows(fn, "out", y)
        ldy = y2.stride(0)
    mean, rstd = _row_stats(x, rows) if stats else (None, None)
    _nfx.check(_lib.nfx_layer_norm(x2.data_ptr(), xt, x2.stride(0), _p(g), _p(b), pt, rows, d, eps, y2.data_ptr(), ldy,
                                   _p(mean), _p(rstd), _stream(x)))
    return (y, mean, rstd) if stats else y


def layer_norm_fp8(x, gamma=None, beta=None, eps=1e-5, stats=False, stream=None):
    """layer_norm(x) in FP8 groups of 128 (Fp8Blocks over the flattened rows): what fp8_quantise
    makes of an fp32 y, which is never written.  With `stats`: (blocks, mean, rstd)."""
    fn = "layer_norm_fp8"
    x2, xt, g, b, pt = _norm_args(fn, x, gamma, beta)
    if _elsewhere(x, stream):
        with _on(x, stream):
            return layer_norm_fp8(x, gamma, beta, eps, stats)
    rows, d = x2.shape
    codes, scales = _codes(rows, d, x.device), _scales(rows, d, x.device)
    mean, rstd = _row_stats(x, rows) if stats else (None, None)
    _nfx.check(_lib.nfx_layer_norm_fp8(x2.data_ptr(), xt, x2.stride(0), _p(g), _p(b), pt, rows, d, eps, codes.data_ptr(),
                                       codes.stride(0), scales.data_ptr(), 1, rows, _p(mean), _p(rstd), _stream(x)))
    q = Fp8Blocks(codes, scales)
    return (q, mean, rstd) if stats else q


def layer_norm_backward(dy, x, mean, rstd, gamma=None, param_grads=True, stream=None):
    """Gradients of layer_norm from dy (of x's shape and type) and the saved fp32 mean and rstd:
    (dx, dgamma, dbeta), the last two in gamma's type (fp32 without gamma), or None without
    `param_grads`."""
    fn = "layer_norm_backward"
    x2, xt, g, _, pt = _norm_args(fn, x, gamma, None)
    rows, d = x2.shape
    if _type(fn, "dy", dy) != xt or dy.shape != x.shape:
        _refuse(fn, "dy must have x's shape and type")
    dy2 = _rows(fn, "dy", dy)
    for name, t in (("mean", mean), ("rstd", rstd)):
        if _type(fn, name, t) != 0 or t.numel() != rows or not t.is_contiguous():
            _refuse(fn, f"{name} must be a contiguous float32 tensor of {rows}")
    _same_device(fn, x, dy=dy, mean=mean, rstd=rstd)
    if _elsewhere(x, stream):
        with _on(x, stream):
            return layer_norm_backward(dy, x, mean, rstd, gamma, param_grads)
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    dg = db = ws = None
    n = 0
    if param_grads:
        dg, db = torch.empty((2, d), dtype=torch.float32 if g is None else g.dtype, device=x.device).unbind(0)
        n = _lib.nfx_layer_norm_backward_workspace(rows, d)
        ws = torch.empty(n, dtype=torch.uint8, device=x.device)
    _nfx.check(_lib.nfx_layer_norm_backward(dy2.data_ptr(), dy2.stride(0), x2.data_ptr(), x2.stride(0), xt, mean.data_ptr(),
                                            rstd.data_ptr(), _p(g), pt, rows, d, dx.data_ptr(), d, _p(dg), _p(db), _p(ws),
                                            n, _stream(x)))
    return dx, dg, db


def fp8_quantise(x, tile=False, transposed=False, col_sums=False, stream=None):
    """x (..., cols), seen as (rows, cols), in FP8: groups of 128 along the rows, or 128 x 128 tiles
    (`tile`, the form for weights).  With `transposed` also the FP8 form of the transpose, from the
    same read of x: its groups run along the rows of x, its tiles have the same codes.  With
    `col_sums` (without `tile`) also the fp32 sums of x's columns.  Returns Fp8Blocks, or a tuple of
    it and what was asked for, in that order."""
    fn = "fp8_quantise"
    xt = _type(fn, "x", x)
    x2 = _rows(fn, "x", x)
    rows, cols = x2.shape
    if tile and col_sums:
        _refuse(fn, "column sums are made with groups of 1 x 128 only")
    if _elsewhere(x, stream):
        with _on(x, stream):
            return fp8_quantise(x, tile, transposed, col_sums)
    dev = x.device
    srows, scols = (-(-rows // GROUP), -(-cols // GROUP)) if tile else (rows, cols)
    codes, scales = _codes(rows, cols, dev), _scales(srows, cols, dev)
    q = Fp8Blocks(codes, scales, tile)
    t = (None, 0, None, 0, 0)
    if transposed:
        ct, st = _codes(cols, rows, dev), _scales(scols, rows, dev)
        t = (ct.data_ptr(), ct.stride(0), st.data_ptr(), 1, scols)
    sums = ws = None
    n = 0
    if col_sums:
        sums = torch.empty(cols, dtype=torch.float32, device=dev)
        n = _lib.nfx_fp8_quantise_workspace(rows, cols)
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
    _nfx.check(_lib.nfx_fp8_quantise(x2.data_ptr(), xt, x2.stride(0), rows, cols, int(tile), codes.data_ptr(),
                                     codes.stride(0), scales.data_ptr(), 1, srows, *t, _p(sums), _p(ws), n, _stream(x)))
    if not (transposed or col_sums):
        return q
    return (q,) + ((Fp8Blocks(ct, st, tile),) if transposed else ()) + ((sums,) if col_sums else ())


def _operand(fn, name, q):
    if not isinstance(q, Fp8Blocks):
        _refuse(fn, f"{name} must be an Fp8Blocks")
    c, s = q.codes, q.scales
    if not c.is_cuda or c.dtype not in (E4M3, torch.uint8) or c.dim() != 2:
        _refuse(fn, f"the codes of {name} must be a 2-D CUDA tensor of float8_e4m3fn (or its bytes)")
    r, k = c.shape
    if k > 1 and c.stride(1) != 1:
        _refuse(fn, f"the last dimension of {name}'s codes must be contiguous")
    want = (_up(r, GROUP) // GROUP if q.tile else r, _up(k, GROUP) // GROUP)
    if not s.is_cuda or s.dtype != torch.float32 or s.shape != want or s.device != c.device:
        _refuse(fn, f"the scales of {name} must be float32 {want} on {c.device}, not {s.dtype} {tuple(s.shape)}")
    return r, k


def fp8_gemm(a, b, bias=None, act=0, out_dtype=torch.bfloat16, out=None, stream=None):
    """act(a b^T + bias) for Fp8Blocks a (M, K) and b (N, K): C (M, N) in `out_dtype`, or in `out` (its
    type; any row stride).  bias (N,) or None; act 0 none, 1 GELU (tanh form), 2 ReLU."""
    fn = "fp8_gemm"
    (m, k), (n, kb) = _operand(fn, "a", a), _operand(fn, "b", b)
    if k != kb:
        _refuse(fn, f"a has {k} columns and b {kb}")
    ac, bc, sa, sb = a.codes, b.codes, a.scales, b.scales
    bias = _vector(fn, "bias", bias, n)
    _same_device(fn, ac, b=bc, bias=bias, out=out)
    if out is None and out_dtype not in _TYPES:
        _refuse(fn, f"out_dtype must be float32, bfloat16 or float16, not {out_dtype}")
    if _elsewhere(ac, stream):
        with _on(ac, stream):
            return fp8_gemm(a, b, bias, act, out_dtype, out)
    if out is None:
        c = torch.empty((m, n), dtype=out_dtype, device=ac.device)
        ct, ldc = _TYPES[out_dtype], n
    else:
        c = out
        ct = _type(fn, "out", c)
        if c.shape != (m, n):
            _refuse(fn, f"out must be ({m}, {n})")
        ldc = _rows(fn, "out", c).stride(0)
    _nfx.check(_lib.nfx_fp8_gemm(ac.data_ptr(), ac.stride(0), sa.data_ptr(), sa.stride(0), sa.stride(1), int(a.tile),
                                 bc.data_ptr(), bc.stride(0), sb.data_ptr(), sb.stride(0), sb.stride(1), int(b.tile), m, n, k,
                                 _p(bias), 0 if bias is None else _TYPES[bias.dtype], int(act), c.data_ptr(), ct, ldc,
                                 _stream(ac)))
    return c


# ---- autograd -------------------------------------------------------------------------------
class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, eps):
        y, mean, rstd = layer_norm(x, gamma, beta, eps, stats=True)
        ctx.save_for_backward(x, gamma, mean, rstd)
        ctx.beta = None if beta is None else beta.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        x, gamma, mean, rstd = ctx.saved_tensors
        params = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dx, dg, db = layer_norm_backward(dy.contiguous(), x, mean, rstd, gamma, param_grads=params)
        return (dx, dg if ctx.needs_input_grad[1] else None,
                db.to(ctx.beta) if ctx.needs_input_grad[2] else None, None)


def layer_norm_autograd(x, gamma=None, beta=None, eps=1e-5):
    """layer_norm as a differentiable function of x, gamma and beta."""
    return _LayerNorm.apply(x, gamma, beta, eps)


class _Fp8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b):
        x2 = _rows("fp8_linear", "x", x, w.shape[1])
        need_dx, need_dw = ctx.needs_input_grad[:2]
        xq, xt = fp8_quantise(x2, transposed=True) if need_dw else (fp8_quantise(x2), None)
        wq, wt = fp8_quantise(w, tile=True, transposed=True) if need_dx else (fp8_quantise(w, tile=True), None)
        ctx.saved = (xt, wt)
        ctx.like = (x.shape, x.dtype, w.dtype, None if b is None else b.dtype)
        return fp8_gemm(xq, wq, bias=b, out_dtype=x.dtype).view(*x.shape[:-1], w.shape[0])

    @staticmethod
    def backward(ctx, dy):
        (xt, wt), (shape, xdt, wdt, bdt) = ctx.saved, ctx.like
        need_dx, need_dw, need_db = ctx.needs_input_grad
        dy = dy.reshape(-1, dy.shape[-1]).contiguous()
        dx = dw = db = None
        # one read of dy makes the operands of both products and the bias gradient
        got = fp8_quantise(dy, transposed=need_dw, col_sums=need_db)
        got = list(got) if need_dw or need_db else [got]
        dq = got.pop(0)
        if need_dw:
            dw = fp8_gemm(got.pop(0), xt, out_dtype=wdt)
        if need_db:
            db = got.pop(0).to(bdt)
        if need_dx:
            dx = fp8_gemm(dq, wt, out_dtype=xdt).view(shape)
        return dx, dw, db


def fp8_linear(x, weight, bias=None):
    """x weight^T + bias with both products' operands in FP8, differentiable: x (..., K) in groups of
    128 along K, weight (N, K) in 128 x 128 tiles; the gradient dy in groups along N for dx and, with x,
    in groups along the tokens for the weight gradient.  Gradients pass through the rounding to FP8
    unchanged; they come in the types of x, weight and bias, the output in x's."""
    fn = "fp8_linear"
    _type(fn, "x", x)
    _type(fn, "weight", weight)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        _refuse(fn, f"weight must be (N, {x.shape[-1] if x.dim() else '?'})")
    _vector(fn, "bias", bias, weight.shape[0])
    _same_device(fn, x, weight=weight, bias=bias)
    return _Fp8Linear.apply(x, weight, bias)
