"""Root-mean-square norm with the residual's addition (csrc/norm.cu).

A block of the model computes ``h = residual + branch`` and norms ``h`` for the
next branch.  ``add_rms_norm`` does both, and the cast to the projections' type,
in one pass over the stream, with gradients for all three inputs;
``add_rms_norm_fp8`` gives the normed rows in 8 bits with scales, for projections
that take 8-bit operands (inference only).

All functions take CUDA tensors of bf16 or fp32 in any combination, any leading
dimensions, and a last dimension D that is a multiple of 8, at most 16384.
Outputs are on the inputs' device, computed on its current stream.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .library import ops as _ops


class _RmsNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, out_dtype):
        y, rstd = _ops.rms_norm(x, weight, eps, out_dtype)
        ctx.save_for_backward(x, weight, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dx, dw = _ops.rms_norm_bwd(dy, *ctx.saved_tensors)
        return dx, dw, None, None


class _AddRmsNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps, out_dtype):
        y, h, rstd = _ops.add_rms_norm(x, residual, weight, eps, out_dtype)
        ctx.save_for_backward(h, weight, rstd)
        ctx.x_dtype = x.dtype
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        if dy is None:                           # only the stream's new value was used
            return (None if dh is None else dh.to(ctx.x_dtype)), dh, None, None, None
        dx, dres, dw = _ops.add_rms_norm_bwd(dy, dh, *ctx.saved_tensors, ctx.x_dtype)
        return dx, dres, dw, None, None


def _eager(name: str, *args):
    """The C++ call of this name, or None where it is not a case for it: while a
    compiler traces, and for tensors that it does not take."""
    return None if torch.compiler.is_compiling() else getattr(_native.eager(), name)(*args)


def _out_dtype(out_dtype: torch.dtype | None, x: torch.Tensor) -> torch.dtype:
    if out_dtype == torch.float8_e4m3fn:
        raise ValueError("rms_norm: an 8-bit output is nothing without its scales: rms_norm_fp8, add_rms_norm_fp8")
    return out_dtype or x.dtype


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, out_dtype: torch.dtype | None = None):
    """x * (mean(x^2) + eps)^-1/2 * weight over the last dimension, in fp32, rounded
    once to out_dtype (default: x's type).  Differentiable in x and weight."""
    y = _eager("rms_norm", x, weight, eps, out_dtype)
    if y is not None:
        return y
    return _RmsNormFn.apply(x, weight, float(eps), _out_dtype(out_dtype, x))


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
                 out_dtype: torch.dtype | None = None):
    """(y, h): h = x + residual rounded to the residual's type, y = rms_norm(h) in
    out_dtype (default: x's type).  The norm is that of h as stored.  Differentiable
    in x, residual and weight."""
    out = _eager("add_rms_norm", x, residual, weight, eps, out_dtype)
    if out is not None:
        return out
    return _AddRmsNormFn.apply(x, residual, weight, float(eps), _out_dtype(out_dtype, x))


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, group: int = 0):
    """(q, scale): rms_norm in float8_e4m3fn.  With group 0 one fp32 scale per row,
    (..., 1); with group 128 one per 128 columns, (..., ceil(D / 128)).  q * scale is
    the norm; the largest magnitude of a group has the code 448.  Has no gradient: a
    backward through it raises."""
    out = _eager("rms_norm_fp8", x, weight, eps, group)
    if out is not None:
        return out
    return _ops.rms_norm_fp8(x, weight, float(eps), group)


def add_rms_norm_fp8(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
                     group: int = 0):
    """(q, scale, h): rms_norm_fp8 of h = x + residual, h in the residual's type.
    Has no gradient: a backward through it raises."""
    out = _eager("add_rms_norm_fp8", x, residual, weight, eps, group)
    if out is not None:
        return out
    return _ops.add_rms_norm_fp8(x, residual, weight, float(eps), group)
