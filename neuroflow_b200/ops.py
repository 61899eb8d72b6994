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
(a torch.cuda.Stream or raw handle), without synchronising; outputs are allocated for that stream.  There is
no CPU fallback.  Refused arguments raise NfxError with code 1 (InvalidArg).  torch.float32, bfloat16 and
float16 are accepted where a tensor is not FP8; the last dimension has to be contiguous.

With `stream` the caller orders it behind the work that made the inputs, and other streams behind it where
they read the outputs (torch.cuda.Stream.wait_stream).  The tensors of the call are recorded on a
torch.cuda.Stream, so they may be released at once; the life of a raw handle's or ExternalStream's stream is
not known to torch, so there the caller keeps them until the work is done.

Codes are float8_e4m3fn by the library's encoder: as torch's conversion rounds, save that a scaled value
under 2^-6, the smallest normal number, is at most 7 * 2^-9, the largest subnormal one (torch gives 2^-6 from
7.5 * 2^-9 on); values beyond +-448 saturate.

Only layer_norm_autograd and fp8_linear are recorded by autograd; the other calls are the operators
themselves, and write into an `out` as torch's own in-place operations do (its version is raised, it must
not require grad while gradients are recorded).
"""
from __future__ import annotations

import contextlib
from typing import NamedTuple

import torch

from . import _nfx  # the library itself, with a clear message where it has not been built

try:
    from . import _nfx_torch as _ext
except ImportError as e:
    raise ImportError("the torch front-end _nfx_torch.so is missing or was built for another torch: build it "
                      "(python -m neuroflow_b200.build, or __graft_entry__.build())") from e

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
def _on(stream, t, *others):
    """`stream` (a torch.cuda.Stream or raw handle on t's device) made current, so that what a call
    allocates belongs to it; the tensors of the call (t, and the others that are not None) are recorded
    on a stream of torch's, so that their memory is not handed out again before it is done with them."""
    if not t.is_cuda:
        _refuse("stream", "the tensors of a call must be CUDA tensors")
    ours = isinstance(stream, torch.cuda.Stream) and not isinstance(stream, torch.cuda.ExternalStream)
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(int(stream), device=t.device)
    elif stream.device != t.device:
        _refuse("stream", f"the stream is on {stream.device}, the tensors are on {t.device}")
    with torch.cuda.stream(stream):
        yield
    if ours:
        for u in (t, *others):
            if u is not None:
                u.record_stream(stream)


def layer_norm(x, gamma=None, beta=None, eps=1e-5, out=None, stats=False, stream=None):
    """Layer norm over the last dimension of x (..., d); gamma and beta (d,), None for ones and
    zeros.  y in x's type (in `out` if given, which may be x); with `stats` also the fp32 mean and 1/std of each
    row, which layer_norm_backward takes: (y, mean, rstd)."""
    if stream is not None:
        with _on(stream, x, gamma, beta, out):
            return _ext.layer_norm(x, gamma, beta, eps, out, stats)
    return _ext.layer_norm(x, gamma, beta, eps, out, stats)


def layer_norm_fp8(x, gamma=None, beta=None, eps=1e-5, stats=False, stream=None):
    """layer_norm(x) in FP8 groups of 128 (Fp8Blocks over the flattened rows): what fp8_quantise
    makes of an fp32 y, which is never written.  With `stats`: (blocks, mean, rstd)."""
    if stream is not None:
        with _on(stream, x, gamma, beta):
            return layer_norm_fp8(x, gamma, beta, eps, stats)
    got = _ext.layer_norm_fp8(x, gamma, beta, eps, stats)
    q = Fp8Blocks(got[0], got[1])
    return (q, got[2], got[3]) if stats else q


def layer_norm_backward(dy, x, mean, rstd, gamma=None, param_grads=True, stream=None):
    """Gradients of layer_norm from dy (of x's shape and type) and the saved fp32 mean and rstd:
    (dx, dgamma, dbeta), the last two in gamma's type (fp32 without gamma), or None without
    `param_grads`."""
    if stream is not None:
        with _on(stream, x, dy, mean, rstd, gamma):
            return _ext.layer_norm_backward(dy, x, mean, rstd, gamma, param_grads)
    return _ext.layer_norm_backward(dy, x, mean, rstd, gamma, param_grads)


def fp8_quantise(x, tile=False, transposed=False, col_sums=False, stream=None):
    """x (..., cols), seen as (rows, cols), in FP8: groups of 128 along the rows, or 128 x 128 tiles
    (`tile`, the form for weights).  With `transposed` also the FP8 form of the transpose, from the
    same read of x: its groups run along the rows of x, its tiles have the same codes.  With
    `col_sums` (without `tile`) also the fp32 sums of x's columns.  Returns Fp8Blocks, or a tuple of
    it and what was asked for, in that order."""
    if stream is not None:
        with _on(stream, x):
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
        with _on(stream, *a[:2], *b[:2], bias, out):
            return _ext.fp8_gemm(*a, *b, bias, act, out_dtype, out)
    return _ext.fp8_gemm(*a, *b, bias, act, out_dtype, out)


# ---- under autograd -------------------------------------------------------------------------
def layer_norm_autograd(x, gamma=None, beta=None, eps=1e-5):
    """layer_norm as a differentiable function of x, gamma and beta (once: differentiating a gradient made
    under create_graph raises, as does a tangent of forward mode)."""
    return _ext.layer_norm_autograd(x, gamma, beta, eps)


def fp8_linear(x, weight, bias=None):
    """x weight^T + bias with both products' operands in FP8, differentiable: x (..., K) in groups of
    128 along K, weight (N, K) in 128 x 128 tiles; the gradient dy in groups along N for dx and, with x,
    in groups along the tokens for the weight gradient.  Gradients pass through the rounding to FP8
    unchanged; they come in the types of x, weight and bias, the output in x's.  Differentiable once:
    differentiating a gradient made under create_graph raises, as does a tangent of forward mode."""
    return _ext.fp8_linear(x, weight, bias)
