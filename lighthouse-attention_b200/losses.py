"""Losses of an output projection whose logits are never stored (csrc/linear_loss.cu).

``linear_cross_entropy(hidden, weight, target)`` is
``F.cross_entropy(hidden @ weight.T, target)`` and ``linear_distillation`` the
divergence from a teacher's top logits, both with gradients for hidden and
weight.  The logits live in tensor memory, tile by tile; the backward forms them
again and goes over the vocabulary in pieces.  Beyond the inputs and the gradients
a call takes, while it runs,

  forward   N V / 16 bytes of statistics (8 bytes per position and 128 entries)
  backward  512 MB of logits' gradients at most (512 N from a million positions
            on), 4 N D bytes of fp32 sums of dhidden, twice that where positions
            are packed, and up to 160 MB of parts of products that are split
  both      a copy of hidden's 2 N D bytes

Between the two a reduced loss over at most 256 entries keeps 512 bytes per
position (the softmax less the targets); otherwise 20 bytes, and 8 per teacher
entry.

hidden (..., D) and weight (V, D) are bf16 CUDA tensors, D a multiple of 8.
Logits, softmax statistics and losses are fp32, gradients bf16.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .library import ops as _ops
from .norm import _eager


class _LinearXentFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, ignore_index, reduction):
        loss, kept = _ops.linear_xent(hidden, weight, target, ignore_index, reduction)
        ctx.save_for_backward(hidden, weight, target, kept)
        ctx.reduction = reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, gout):
        dh, dw = _ops.linear_xent_bwd(*ctx.saved_tensors, gout, ctx.reduction)
        return dh, dw, None, None, None


class _LinearDistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, teacher_logits, teacher_indices, temperature, reduction):
        loss, kept = _ops.linear_distill(hidden, weight, teacher_logits, teacher_indices, temperature, reduction)
        ctx.save_for_backward(hidden, weight, kept)
        ctx.K, ctx.temperature, ctx.reduction = teacher_indices.shape[1], temperature, reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, gout):
        dh, dw = _ops.linear_distill_bwd(*ctx.saved_tensors, gout, ctx.K, ctx.temperature, ctx.reduction)
        return dh, dw, None, None, None, None


def _rows(hidden: torch.Tensor, *per_row: tuple[torch.Tensor, int]):
    """hidden as (N, D); each (tensor, trailing dimensions) must have its leading dimensions."""
    lead = hidden.shape[:-1]
    for t, tail in per_row:
        if t.shape[:t.dim() - tail] != lead:
            raise ValueError(f"leading dimensions {tuple(lead)} of hidden and {tuple(t.shape)} differ")
    return hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1])


def _long(t: torch.Tensor, *shape: int) -> torch.Tensor:
    """t as int64 of this shape."""
    if t.dtype != torch.int64:
        if t.dtype != torch.int32:
            raise ValueError(f"targets and indices must be int64 or int32, got {t.dtype}")
        t = t.to(torch.int64)
    return t if t.shape == shape else t.reshape(shape)


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of the logits ``hidden @ weight.T``.

    target (...) int64 or int32 has hidden's leading dimensions.  Positions with
    target ignore_index have loss 0 and no gradient; any other target outside
    [0, V) makes the position's loss NaN.  reduction "mean" (over the positions
    that are not ignored; 0 where all are), "sum", or "none" (the loss of every
    position).  Returns fp32."""
    h = _rows(hidden, (target, 0))
    target_ = _long(target, h.shape[0])
    loss = _eager("linear_xent", h, weight, target_, ignore_index, _native.REDUCTIONS.get(reduction, -1))
    if loss is None:
        loss = _LinearXentFn.apply(h, weight, target_, ignore_index, reduction)
    return loss.view(target.shape) if reduction == "none" and target.dim() != 1 else loss


def linear_distillation(hidden: torch.Tensor, weight: torch.Tensor, teacher_logits: torch.Tensor,
                        teacher_indices: torch.Tensor, temperature: float = 1.0,
                        reduction: str = "mean") -> torch.Tensor:
    """Divergence of the student ``softmax(hidden @ weight.T / T)`` from a teacher
    known by its top logits.

    teacher_logits (..., K) bf16 or fp32 and teacher_indices (..., K) int64 or
    int32, K at most 256, in any order; a negative index marks an absent entry.
    With p = softmax(teacher_logits / T) over a position's entries, T within
    [1e-18, 1e18], loss = T^2 sum_k p_k (log p_k - log student_k).  A position without entries
    has loss 0, no gradient and does not count in the mean.  Entries with the
    same index add up; an index >= V, or a logit that is NaN or +infinity, makes
    the position's loss NaN.  The teacher gets no gradient.  Returns fp32."""
    h = _rows(hidden, (teacher_logits, 1), (teacher_indices, 1))
    N = h.shape[0]
    tl = teacher_logits if teacher_logits.dim() == 2 else teacher_logits.reshape(N, teacher_logits.shape[-1])
    ti, temperature = _long(teacher_indices, N, teacher_indices.shape[-1]), float(temperature)
    loss = _eager("linear_distill", h, weight, tl, ti, temperature, _native.REDUCTIONS.get(reduction, -1))
    if loss is None:
        loss = _LinearDistillFn.apply(h, weight, tl, ti, temperature, reduction)
    return loss.view(hidden.shape[:-1]) if reduction == "none" and hidden.dim() != 2 else loss
