"""Operators of transformer blocks on CUDA tensors, forward and backward: layer norm, the FP8 E4M3 block
quantiser and the FP8 block-scaled product; RMS norm with the residual's addition, the 16-bit product with
bias, activation and residual, and gradient clipping.

    from neuroflow_b200 import ops
    y, mean, rstd = ops.layer_norm(x, gamma, beta, stats=True)
    dx, dgamma, dbeta = ops.layer_norm_backward(dy, x, mean, rstd, gamma)
    w8 = ops.fp8_quantise(w, tile=True)                  # once per weight
    x8 = ops.layer_norm_fp8(x, gamma, beta)              # layer norm straight into FP8
    y = ops.fp8_gemm(x8, w8, bias=b, act=1)              # act(x8 w8^T + b)
    y = ops.fp8_linear(x, w, b); y.backward(dy)          # the same linear layer under autograd

    n, h = ops.rms_norm(x, gamma, residual=h)            # h = x + h, n = its RMS norm; rms_norm_fp8: n in FP8
    y = ops.gemm(n, w, bias=b, act=1, residual=h)        # act(n w^T + b) + h in bf16 or fp16
    y = ops.linear(n, w, b, act=1, residual=h)           # the same under autograd
    norm = ops.clip_grad_norm([p.grad for p in params], 1.0)

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

Only layer_norm_autograd, fp8_linear, rms_norm_autograd and linear are recorded by autograd; the other calls
are the operators themselves, and write into an `out` as torch's own in-place operations do (its version is
raised, it must not require grad while gradients are recorded).
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


# ---- a block in 16 bits -----------------------------------------------------------------------
def rms_norm(x, gamma=None, eps=1e-5, residual=None, out=None, sum_out=None, stats=False, stream=None):
    """RMS norm over the last dimension of x (..., d): y = h gamma / sqrt(mean(h^2) + eps), with h = x, or
    with a `residual` of x's shape (and type, or float32) h = x + residual in the residual's type; the norm
    is that of h as it is stored.  gamma (d,), None for ones.  y in x's type.  Returns y; (y, h) with a
    residual; with `stats` also the fp32 1 / root mean square of each row, which rms_norm_backward takes, as the
    last one.  `out` receives y and may be x or the residual, `sum_out` receives h and may be the residual or x
    (the very tensor, of the same type)."""
    if stream is not None:
        with _on(stream, x, gamma, residual, out, sum_out):
            return _ext.rms_norm(x, gamma, eps, residual, out, sum_out, stats)
    return _ext.rms_norm(x, gamma, eps, residual, out, sum_out, stats)


def rms_norm_fp8(x, gamma=None, eps=1e-5, residual=None, sum_out=None, stats=False, stream=None):
    """rms_norm with y in FP8 groups of 128 (Fp8Blocks over the flattened rows): what fp8_quantise makes of
    an fp32 y, which is never written.  Returns as rms_norm, with the blocks in y's place."""
    if stream is not None:
        with _on(stream, x, gamma, residual, sum_out):
            return rms_norm_fp8(x, gamma, eps, residual, sum_out, stats)
    codes, scales, h, rstd = _ext.rms_norm_fp8(x, gamma, eps, residual, sum_out, stats)
    got = (Fp8Blocks(codes, scales),) + ((h,) if h is not None else ()) + ((rstd,) if stats else ())
    return got if len(got) > 1 else got[0]


def rms_norm_backward(dy, h, rstd, gamma=None, dsum=None, param_grads=True, stream=None):
    """Gradients of rms_norm from dy (of y's shape and type), the normalised h (rms_norm's sum; x itself where
    there was no residual) and the saved fp32 rstd; `dsum`, of h's type, is the gradient that reaches h from
    elsewhere (the residual stream) and is added.  Returns (dx, dresidual, dgamma): dx in dy's type,
    dresidual in h's (the same tensor where the types are equal: the gradient of x + residual is that of both),
    dgamma in gamma's type (fp32 without gamma), or None without `param_grads`."""
    if stream is not None:
        with _on(stream, h, dy, rstd, gamma, dsum):
            return _ext.rms_norm_backward(dy, h, rstd, gamma, dsum, param_grads)
    return _ext.rms_norm_backward(dy, h, rstd, gamma, dsum, param_grads)


def gemm(a, b, bias=None, act=0, residual=None, out_dtype=None, out=None, preact=False, stream=None):
    """act(a b^T + bias) + residual for a (M, K) and b (N, K), both bfloat16 or both float16, sums in fp32: C
    (M, N) in the operands' type, or in `out_dtype` (that or float32), or in `out` (its type; any row
    stride; it may be the residual).  Rows or columns of a and of b are contiguous: a.t() and b.t() are taken
    as they are.  bias (N,) or None; act 0 none, 1 GELU (tanh form), 2 ReLU; residual (M, N) of C's type.  With
    `preact`: (C, a b^T + bias) of one type, the second for act_backward.  Operands whose base or row
    stride is no multiple of 16 bytes are copied first."""
    if stream is not None:
        with _on(stream, a, b, bias, residual, out):
            return _ext.gemm(a, b, bias, act, residual, out_dtype, out, preact)
    return _ext.gemm(a, b, bias, act, residual, out_dtype, out, preact)


def act_backward(dy, z, act, bias_dtype=None, stream=None):
    """Gradient of act(z): (dz, dbias), dz = dy act'(z) in dy's type (dy itself with act = 0, where z may be
    None); dbias, in `bias_dtype`, the sums of dz over its rows formed in fp32, None without a type."""
    if stream is not None:
        with _on(stream, dy, z):
            return _ext.act_backward(dy, z, act, bias_dtype)
    return _ext.act_backward(dy, z, act, bias_dtype)


def grad_norm(grads, stream=None):
    """The 2-norm over all elements of the tensors `grads` (one device; float32, bfloat16 and float16 may be
    mixed; contiguous, or permutations of contiguous tensors): a float32 tensor without dimensions, on the
    device.  Groups of up to 32 squares (16 of float32 elements) are added in fp32, or in 64 bits where that would
    over- or underflow, and the groups in 64 bits."""
    grads = list(grads)
    if stream is not None and grads:
        with _on(stream, *grads):
            return _ext.grad_norm(grads)
    return _ext.grad_norm(grads)


def clip_grad_norm(grads, max_norm, eps=1e-6, out=None, stream=None):
    """Scales `grads` (as in grad_norm) in place by min(1, max_norm / (norm + eps)) and returns norm, their
    2-norm before, as grad_norm does; nothing is copied to the host.  A norm of infinity makes zeros of finite elements
    and NaN of infinite ones, a max_norm of infinity scales nothing, and a NaN makes NaN of everything.  With `out`, a tensor for each gradient (of
    its shape and any of the three types; it may be the gradient itself), the gradients are left alone and the
    scaled ones go there.  No tensor that is written shares memory with another."""
    grads = list(grads)
    out = None if out is None else list(out)
    if stream is not None and grads:
        with _on(stream, *grads, *(out or ())):
            return _ext.clip_grad_norm(grads, max_norm, eps, out)
    return _ext.clip_grad_norm(grads, max_norm, eps, out)


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


def rms_norm_autograd(x, gamma=None, eps=1e-5, residual=None):
    """rms_norm as a differentiable function of x, gamma and the residual: y, or (y, x + residual); once, as
    layer_norm_autograd."""
    return _ext.rms_norm_autograd(x, gamma, eps, residual)


def linear(x, weight, bias=None, act=0, residual=None):
    """act(x weight^T + bias) + residual, differentiable: x (..., K) and weight (N, K) both bfloat16 or both
    float16, bias (N,) of any type, residual and result (..., N) of x's type.  Gradients come in the types of
    their tensors, sums in fp32; with an activation dz = dy act'(z) is rounded to x's type in between, as is the z
    that is kept for it (gemm with preact and out_dtype float32, and act_backward, keep both in fp32).  Once, as
    fp8_linear."""
    return _ext.linear(x, weight, bias, act, residual)
