"""The post-training losses on top of the tied LM head: ``logits = y @ e^T``, a loss over them, and the
two products of its backward, as one autograd node.

The counterpart of :func:`ferrite.kernels.cross_entropy.tied_head_cross_entropy` for
:mod:`policy_loss`, :mod:`preference_loss` and :mod:`distillation`.  Each of those gives the gradient in the
logits together with the loss, already in the type of the head's products, so the logits are gone before
the backward begins: what is kept for it is the 16-bit gradient, half or a quarter of a set of f32 logits and
their f32 gradient.
"""

from __future__ import annotations

import torch

from ferrite.kernels.distillation import DistillationLoss, distillation_loss_and_grad
from ferrite.kernels.matmul import gemm
from ferrite.kernels.policy_loss import PolicyLoss, policy_loss_and_grad
from ferrite.kernels.preference_loss import PreferenceLoss, preference_loss_and_grad


class _TiedHead(torch.autograd.Function):
    """``loss_and_grad(logits, *args, **kw)`` at ``logits = y e^T``; the gradient in the logits is taken for an
    upstream gradient of 1 and the products' results are scaled by the real one."""

    @staticmethod
    def forward(ctx, y, e, loss_and_grad, args, kw, logits_dtype):
        logits = gemm(y, e, trans_b=True, out_dtype=logits_dtype)
        out, dl = loss_and_grad(logits, *args, grad_dtype=y.dtype, **kw)
        ctx.save_for_backward(y, e, dl)
        ctx.mark_non_differentiable(*out[1:])
        return tuple(out)

    @staticmethod
    def backward(ctx, g, *_):
        y, e, dl = ctx.saved_tensors
        dy = gemm(dl, e, out_dtype=y.dtype).mul_(g) if ctx.needs_input_grad[0] else None
        de = gemm(dl, y, trans_a=True, out_dtype=e.dtype).mul_(g) if ctx.needs_input_grad[1] else None
        return dy, de, None, None, None, None


def _apply(y, e, loss_and_grad, args, kw, logits_dtype):
    if y.ndim != 2 or e.ndim != 2 or y.shape[1] != e.shape[1]:
        raise ValueError(f"expected y [rows, d] and e [vocab, d]; got {tuple(y.shape)} and {tuple(e.shape)}")
    if y.dtype != e.dtype:
        raise ValueError("y and the embedding must share a dtype")
    if logits_dtype not in (torch.float32, y.dtype):
        raise TypeError(f"logits of type {logits_dtype}: expected float32 or {y.dtype}")
    return _TiedHead.apply(y, e, loss_and_grad, args, kw, logits_dtype)


def tied_head_policy_loss(y, e, targets, old_logprobs, advantages, weights=None, *, logits_dtype=torch.float32, **kw) -> PolicyLoss:
    """:func:`ferrite.kernels.policy_loss.policy_loss` of the tied head's logits, differentiable in ``y``
    ``[rows, d]`` and the embedding ``e [vocab, d]``.  ``logits_dtype``: f32, or their own type for half the traffic."""
    return PolicyLoss(*_apply(y, e, policy_loss_and_grad, (targets, old_logprobs, advantages, weights), kw, logits_dtype))


def tied_head_preference_loss(y, e, targets, ref_logprobs, offsets, *, logits_dtype=torch.float32, **kw) -> PreferenceLoss:
    """:func:`ferrite.kernels.preference_loss.preference_loss` of the tied head's logits."""
    return PreferenceLoss(*_apply(y, e, preference_loss_and_grad, (targets, ref_logprobs, offsets), kw, logits_dtype))


def tied_head_distillation_loss(y, e, teacher_values, teacher_indices, weights=None, *, logits_dtype=torch.float32, **kw) -> DistillationLoss:
    """:func:`ferrite.kernels.distillation.distillation_loss` of the tied head's logits."""
    return DistillationLoss(*_apply(y, e, distillation_loss_and_grad, (teacher_values, teacher_indices, weights), kw, logits_dtype))
