"""Operators of one pre-norm FP8 linear layer on CUDA tensors: layer norm, the FP8 E4M3 block
quantiser and the FP8 block-scaled product, forward and backward.

    from neuroflow_b200 import ops
    y, mean, rstd = ops.layer_norm(x, gamma, beta, stats=True)
    dx, dgamma, dbeta = ops.layer_norm_backward(dy, x, mean, rstd, gamma)
    w8 = ops.fp8_quantise(w, tile=True)                  # once per weight
    x8 = ops.layer_norm_fp8(x, gamma, beta)              # layer norm straight into FP8
    y = ops.fp8_gemm(x8, w8, bias=b, act=1)              # act(x8 w8^T + b)
    y = ops.fp8_linear(x, w, b); y.backward(dy)          # the same linear layer under autograd

Every call runs the kernels of libnfx.so (the C-ABI of include/nfx.h, reached through the compiled
front-end torch_ext/nfx_torch.cpp) on the current torch stream of the tensors' device, or on `stream`
(a torch.cuda.Stream or raw handle), without synchronising; outputs are allocated for that stream.  There is no CPU fallback.  Refused
arguments raise NfxError with code 1 (InvalidArg).  torch.float32, bfloat16 and float16 are
accepted where a tensor is not FP8; the last dimension has to be contiguous.
"""
from __future__ import annotations

import contextlib
from typing import NamedTuple

import torch

from . import _nfx  # the library itself, with a clear message where it has not been built
from . import _nfx_torch as _ext

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


@contextlib.contextmanager
def _on(t, stream):
    """`stream` (a torch.cuda.Stream or raw handle on t's device) made current, so that what a call
    allocates belongs to it."""
    if not t.is_cuda:
        _refuse("stream", "the tensors of a call must be CUDA tensors")
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(int(stream), device=t.device)
    with torch.cuda.stream(stream):
        yield


def layer_norm(x, gamma=None, beta=None, eps=1e-5, out=None, stats=False, stream=None):
    """Layer norm over the last dimension of x (..., d); gamma and beta (d,), None for ones and
    zeros.  y in x's type (in `out` if given); with `stats` also the fp32 mean and 1/std of each
    row, which layer_norm_backward takes: (y, mean, rstd)."""
    if stream is not None:
        with _on(x, stream):
            return _ext.layer_norm(x, gamma, beta, eps, out, stats)
    return _ext.layer_norm(x, gamma, beta, eps, out, stats)


def layer_norm_fp8(x, gamma=None, beta=None, eps=1e-5, stats=False, stream=None):
    """layer_norm(x) in FP8 groups of 128 (Fp8Blocks over the flattened rows): what fp8_quantise
    makes of an fp32 y, which is never written.  With `stats`: (blocks, mean, rstd)."""
    if stream is not None:
        with _on(x, stream):
            return layer_norm_fp8(x, gamma, beta, eps, stats)
    got = _ext.layer_norm_fp8(x, gamma, beta, eps, stats)
    q = Fp8Blocks(got[0], got[1])
    return (q, got[2], got[3]) if stats else q


def layer_norm_backward(dy, x, mean, rstd, gamma=None, param_grads=True, stream=None):
    """Gradients of layer_norm from dy (of x's shape and type) and the saved fp32 mean and rstd:
    (dx, dgamma, dbeta), the last two in gamma's type (fp32 without gamma), or None without
    `param_grads`."""
    if stream is not None:
        with _on(x, stream):
            return _ext.layer_norm_backward(dy, x, mean, rstd, gamma, param_grads)
    return _ext.layer_norm_backward(dy, x, mean, rstd, gamma, param_grads)


def fp8_quantise(x, tile=False, transposed=False, col_sums=False, stream=None):
    """x (..., cols), seen as (rows, cols), in FP8: groups of 128 along the rows, or 128 x 128 tiles
    (`tile`, the form for weights).  With `transposed` also the FP8 form of the transpose, from the
    same read of x: its groups run along the rows of x, its tiles have the same codes.  With
    `col_sums` (without `tile`) also the fp32 sums of x's columns.  Returns Fp8Blocks, or a tuple of
    it and what was asked for, in that order."""
    if stream is not None:
        with _on(x, stream):
            return fp8_quantise(x, tile, transposed, col_sums)
    codes, scales, other, sums = _ext.fp8_quantise(x, tile, transposed, col_sums)
    q = Fp8Blocks(codes, scales, tile)
    if not (transposed or col_sums):
        return q
    return (q,) + ((Fp8Blocks(*other, tile),) if transposed else ()) + ((sums,) if col_sums else ())


def fp8_gemm(a, b, bias=None, act=0, out_dtype=torch.bfloat16, out=None, stream=None):
    """act(a b^T + bias) for Fp8Blocks a (M, K) and b (N, K): C (M, N) in `out_dtype`, or in `out` (its
    type; any row stride).  bias (N,) or None; act 0 none, 1 GELU (tanh form), 2 ReLU."""
    if not (isinstance(a, Fp8Blocks) and isinstance(b, Fp8Blocks)):
        _refuse("fp8_gemm", "a and b must be Fp8Blocks")
    if stream is not None:
        with _on(a.codes, stream):
            return _ext.fp8_gemm(*a, *b, bias, act, out_dtype, out)
    return _ext.fp8_gemm(*a, *b, bias, act, out_dtype, out)


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
        need_dx, need_dw = ctx.needs_input_grad[:2]
        xq, xt = fp8_quantise(x, transposed=True) if need_dw else (fp8_quantise(x), None)
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
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        _refuse("fp8_linear", f"weight must be (N, {x.shape[-1] if x.dim() else '?'})")
    if bias is not None and bias.shape != weight.shape[:1]:
        _refuse("fp8_linear", f"bias must be a vector of {weight.shape[0]}")
    return _Fp8Linear.apply(x, weight, bias)
