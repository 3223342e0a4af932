"""The post-training losses on top of the tied LM head: ``logits = y @ e^T``, a loss over them, and the
two products of its backward, as one autograd node.

The counterpart of :func:`ferrite.kernels.cross_entropy.tied_head_cross_entropy` for
:mod:`policy_loss`, :mod:`preference_loss` and :mod:`distillation`.  Each of those gives the gradient in the
logits together with the loss, already in the type of the head's products.  With bf16 (and f32) operands the logits are
therefore gone before the backward begins: what is kept for it is the gradient for an upstream gradient of 1, which
has f32's range, and the products' results are scaled by the real one.  f16 has too few exponents for
that -- a row's share of a mean over thousands of rows, times a probability, is 0 there -- so with f16 operands the
logits are kept, and the gradient is taken in the backward, with the real upstream gradient (a loss scale) in it
before it is rounded.
"""

from __future__ import annotations

import torch

from ferrite.kernels import _rows
from ferrite.kernels.distillation import DistillationLoss, distillation_loss, distillation_loss_and_grad
from ferrite.kernels.matmul import gemm
from ferrite.kernels.policy_loss import PolicyLoss, policy_loss, policy_loss_and_grad
from ferrite.kernels.preference_loss import PreferenceLoss, preference_loss, preference_loss_and_grad


class _TiedHead(torch.autograd.Function):
    """``loss_and_grad(logits, *args, **kw)`` at ``logits = y e^T``: the gradient in the logits is taken for an
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
        dy, de = (_rows.first_only(d if d is None else d.mul_(g), y, e, g) for d in _products(ctx, dl, y, e))
        return dy, de, None, None, None, None


class _TiedHeadLate(torch.autograd.Function):
    """The same with the gradient in the logits taken in the backward, for the real upstream gradient."""

    @staticmethod
    def forward(ctx, y, e, loss, loss_and_grad, kw, logits_dtype, *args):
        logits = gemm(y, e, trans_b=True, out_dtype=logits_dtype)
        named = [k for k, v in kw.items() if isinstance(v, torch.Tensor)]
        out = loss(logits, *args, **kw)
        ctx.save_for_backward(y, e, logits, *(kw[k] for k in named), *args)
        ctx.loss_and_grad, ctx.named, ctx.kw = loss_and_grad, named, {k: v for k, v in kw.items() if k not in named}
        ctx.mark_non_differentiable(*out[1:])
        return tuple(out)

    @staticmethod
    def backward(ctx, g, *_):
        y, e, logits, *rest = ctx.saved_tensors
        n = len(ctx.named)
        _, dl = ctx.loss_and_grad(logits, *rest[n:], grad_dtype=y.dtype, upstream=g, **dict(zip(ctx.named, rest[:n])), **ctx.kw)
        dy, de = (_rows.first_only(d, y, e, g) for d in _products(ctx, dl, y, e))
        return (dy, de, *([None] * (len(rest) - n + 4)))


def _products(ctx, dl, y, e):
    dy = gemm(dl, e, out_dtype=y.dtype) if ctx.needs_input_grad[0] else None
    de = gemm(dl, y, trans_a=True, out_dtype=e.dtype) if ctx.needs_input_grad[1] else None
    return dy, de


def _apply(y, e, loss, loss_and_grad, args, kw, logits_dtype):
    for name in ("grad_scale", "grad_dtype", "upstream"):
        if name in kw:
            raise TypeError(f"{name} is of the logits' own gradient; the gradients of y and the embedding are autograd's")
    if y.ndim != 2 or e.ndim != 2 or y.shape[1] != e.shape[1]:
        raise ValueError(f"expected y [rows, d] and e [vocab, d]; got {tuple(y.shape)} and {tuple(e.shape)}")
    if y.dtype != e.dtype:
        raise ValueError("y and the embedding must share a dtype")
    if logits_dtype not in (torch.float32, y.dtype):
        raise TypeError(f"logits of type {logits_dtype}: expected float32 or {y.dtype}")
    if not _rows.recorded(y, e):  # an evaluation: the loss alone
        with torch.no_grad():
            return loss(gemm(y, e, trans_b=True, out_dtype=logits_dtype), *args, **kw)
    if any(isinstance(t, torch.Tensor) and t.requires_grad for t in (*args, *kw.values())):
        raise ValueError("an argument requires a gradient, but the loss is differentiable in y and the embedding only: pass it detached")
    if y.dtype == torch.float16:
        return _TiedHeadLate.apply(y, e, loss, loss_and_grad, kw, logits_dtype, *args)
    return _TiedHead.apply(y, e, loss_and_grad, args, kw, logits_dtype)


def tied_head_policy_loss(y, e, targets, old_logprobs, advantages, weights=None, *, logits_dtype=torch.float32, **kw) -> PolicyLoss:
    """:func:`ferrite.kernels.policy_loss.policy_loss` of the tied head's logits, differentiable in ``y``
    ``[rows, d]`` and the embedding ``e [vocab, d]``.  ``logits_dtype``: f32, or their own type for half the traffic."""
    return PolicyLoss(*_apply(y, e, policy_loss, policy_loss_and_grad, (targets, old_logprobs, advantages, weights), kw, logits_dtype))


def tied_head_preference_loss(y, e, targets, ref_logprobs, offsets, *, logits_dtype=torch.float32, **kw) -> PreferenceLoss:
    """:func:`ferrite.kernels.preference_loss.preference_loss` of the tied head's logits."""
    return PreferenceLoss(*_apply(y, e, preference_loss, preference_loss_and_grad, (targets, ref_logprobs, offsets), kw, logits_dtype))


def tied_head_distillation_loss(y, e, teacher_values, teacher_indices, weights=None, *, logits_dtype=torch.float32, **kw) -> DistillationLoss:
    """:func:`ferrite.kernels.distillation.distillation_loss` of the tied head's logits."""
    return DistillationLoss(*_apply(y, e, distillation_loss, distillation_loss_and_grad, (teacher_values, teacher_indices, weights), kw, logits_dtype))
