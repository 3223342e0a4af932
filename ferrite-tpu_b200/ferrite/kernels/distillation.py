"""Distillation from a teacher's top logits, over student logits ``[rows, vocab]``.

A teacher's output is kept as lists of its best tokens and their logits, ``[rows, top]``::

    q    = softmax(teacher_values / temperature) over the row's list
    KL   = sum_j q_j (log q_j - log p[teacher_indices_j]),   p = softmax(logits / temperature)
    loss = sum_r weights_r temperature^2 KL_r

Loss and gradient come from one launch (``ferrite_distill_loss``).  An entry with a negative
index, or the value -inf, is absent; a row without entries is masked.  No counterpart in the
reference, whose only loss is the mean cross-entropy (src/ferrite/model/gpt.py:147-152).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ferrite import _native as nat
from ferrite.kernels import _rows

MAX_TOP = 1024


class DistillationLoss(NamedTuple):
    loss: torch.Tensor  # f32 scalar
    per_token: torch.Tensor  # f32 [rows]: temperature^2 KL; zeros for masked rows


def _check(logits, teacher_values, teacher_indices, weights, temperature, grad_dtype):
    rows, _ = _rows.check_logits(logits, grad_dtype)
    if teacher_values.ndim != 2 or teacher_values.shape != teacher_indices.shape or teacher_values.shape[0] != rows:
        raise ValueError(f"teacher lists must both be [{rows}, top], got {tuple(teacher_values.shape)} and {tuple(teacher_indices.shape)}")
    if not 1 <= teacher_values.shape[1] <= MAX_TOP:
        raise ValueError(f"lists of 1 to {MAX_TOP} entries are supported, got {teacher_values.shape[1]}")
    if teacher_indices.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"teacher_indices must be int32 or int64, got {teacher_indices.dtype}")
    nat.dtype_code(teacher_values.dtype)
    weights = _rows.per_row(weights, rows, "weights")
    _rows.same_device(logits, teacher_values, teacher_indices, weights)
    return teacher_values.detach().contiguous(), teacher_indices.contiguous(), weights, _rows.check_temperature(temperature)


def _launch(logits, values, indices, weights, temperature, grad_dtype, dloss, grad_scale):
    rows, vocab = logits.shape
    top, dev = values.shape[1], logits.device
    loss = torch.empty((), dtype=torch.float32, device=dev)
    f = torch.empty((2, rows), dtype=torch.float32, device=dev)  # per-token losses and the terms of the sum
    base = f.data_ptr()
    grad = None if grad_dtype is None else _rows.empty_grad(logits, grad_dtype)
    nat.check(
        nat.lib().ferrite_distill_loss(
            nat.stream_ptr(dev), logits.data_ptr(), values.data_ptr(), indices.data_ptr(), nat.ptr(weights), temperature, nat.ptr(dloss),
            grad_scale, loss.data_ptr(), base, nat.ptr(grad), base + 4 * rows, 4 * rows, rows, vocab, top, _rows.row_stride(logits),
            vocab if grad is None else _rows.row_stride(grad), top, nat.dtype_code(logits.dtype), nat.dtype_code(values.dtype), int(indices.dtype == torch.int64),
            -1 if grad_dtype is None else nat.dtype_code(grad_dtype),
        )
    )
    return DistillationLoss(loss, f.unbind()[0]), grad


class _Distillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, values, indices, weights, temperature):
        out, _ = _launch(logits, values, indices, weights, temperature, None, None, 1.0)
        ctx.save_for_backward(logits, values, indices, weights)
        ctx.temperature = temperature
        ctx.mark_non_differentiable(out.per_token)
        return tuple(out)

    @staticmethod
    @nat.on_tensor_device
    def backward(ctx, g, *_):
        # statistics and gradient in one launch, as in the policy loss
        logits, values, indices, weights = ctx.saved_tensors
        _, grad = _launch(logits, values, indices, weights, ctx.temperature, logits.dtype, _rows.upstream(g, logits), 1.0)
        return _rows.first_only(grad, logits, g), None, None, None, None


@nat.on_tensor_device
def distillation_loss(logits, teacher_values, teacher_indices, weights=None, *, temperature: float = 1.0) -> DistillationLoss:
    """The distillation loss of ``logits [rows, vocab]`` against lists of a teacher's best tokens (see the
    top of this file); ``loss`` is differentiable in the logits alone.

    teacher_values: ``[rows, top]`` f32, bf16 or f16 logits; teacher_indices: int32 or int64 tokens (an
    index at or above the vocabulary gives NaN; a token listed twice counts with both weights), at most
    1024 a row.  weights: one for each row, ``1 / rows`` by default; a row of weight zero is not read and
    gives zeros.
    """
    recorded = _rows.differentiable(logits, teacher_values=teacher_values, weights=weights)
    values, indices, weights, temperature = _check(logits, teacher_values, teacher_indices, weights, temperature, None)
    if not recorded:
        return _launch(logits, values, indices, weights, temperature, None, None, 1.0)[0]
    return DistillationLoss(*_Distillation.apply(logits, values, indices, weights, temperature))


@nat.on_tensor_device
def distillation_loss_and_grad(logits, teacher_values, teacher_indices, weights=None, *, temperature: float = 1.0, grad_scale: float = 1.0,
                               grad_dtype=None, upstream: torch.Tensor | None = None) -> tuple[DistillationLoss, torch.Tensor]:
    """:func:`distillation_loss` and ``grad_scale`` times its gradient in the logits, in one pass over
    them; ``grad_dtype`` defaults to the logits' type (f32 logits also give bf16 or f16).  ``upstream``, a scalar
    on the device, multiplies the gradient as well, before it is rounded."""
    grad_dtype = grad_dtype or logits.dtype
    values, indices, weights, temperature = _check(logits, teacher_values, teacher_indices, weights, temperature, grad_dtype)
    dloss = None if upstream is None else _rows.upstream(upstream, logits)
    return _launch(logits, values, indices, weights, temperature, grad_dtype, dloss, float(grad_scale))


def distillation_loss_reference(logits, teacher_values, teacher_indices, weights=None, *, temperature=1.0) -> DistillationLoss:
    """The same in plain torch f32, differentiable (the definition the kernels are checked against)."""
    rows = logits.shape[0]
    w = torch.full((rows,), 1.0 / max(rows, 1), device=logits.device) if weights is None else weights.float()
    v = teacher_values.float()
    there = (teacher_indices >= 0) & (v > -float("inf"))
    live = (w != 0) & there.any(1)
    v = torch.where(there & live[:, None], v / temperature, -float("inf"))
    logq = torch.log_softmax(torch.where(live[:, None], v, 0.0), dim=1)
    q = torch.where(there & live[:, None], logq.exp(), 0.0)
    logp = torch.log_softmax(logits.float() / temperature, dim=1).gather(1, torch.where(there, teacher_indices, 0).long())
    kl = torch.where(q > 0, q * (torch.where(q > 0, logq, 0.0) - torch.where(q > 0, logp, 0.0)), 0.0).sum(1) * temperature**2
    kl = torch.where(live, kl, 0.0)
    return DistillationLoss((torch.where(live, w, 0.0) * kl).sum(), kl.detach())
