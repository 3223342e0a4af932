"""The clipped policy loss with a KL term and an entropy bonus, over logits ``[rows, vocab]``.

For the token ``t_r`` written at row ``r``, with ``logp_r`` its log-probability under ``logits /
temperature`` and ``H_r`` the row's entropy::

    ratio = exp(logp - old_logprobs)
    pg    = -min(ratio A, clamp(ratio, 1 - clip_low, 1 + clip_high) A)
    kl    = exp(ref - logp) - (ref - logp) - 1            (an unbiased estimate of KL(p || ref), never negative)
    loss  = sum_r weights_r (pg_r + kl_coef kl_r - entropy_coef H_r)

Loss and gradient come from one launch (``ferrite_policy_loss``): a row's coefficient needs
nothing but the row, so the gradient is written while the row is at hand.  No counterpart in
the reference, whose only loss is the mean cross-entropy (src/ferrite/model/gpt.py:147-152).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ferrite import _native as nat
from ferrite.kernels import _rows
from ferrite.kernels._rows import IGNORE_INDEX


class PolicyLoss(NamedTuple):
    loss: torch.Tensor  # f32 scalar
    logprobs: torch.Tensor  # f32 [rows]; zeros for masked rows, as the three below
    entropy: torch.Tensor  # f32 [rows]
    kl: torch.Tensor  # f32 [rows]; zeros without ref_logprobs
    clipped: torch.Tensor  # bool [rows]: the clipped branch is the smaller


def _check(logits, targets, old_logprobs, advantages, weights, ref_logprobs, clip_low, clip_high, temperature, grad_dtype):
    rows, _ = _rows.check_logits(logits, grad_dtype)
    targets, _ = _rows.check_targets(targets, rows)
    if not (clip_low >= 0.0 and clip_high >= 0.0):
        raise ValueError(f"clip_low and clip_high must not be negative, got {clip_low} and {clip_high}")
    rest = [_rows.per_row(t, rows, n) for t, n in ((old_logprobs, "old_logprobs"), (advantages, "advantages"), (weights, "weights"), (ref_logprobs, "ref_logprobs"))]
    _rows.same_device(logits, targets, *rest)
    return targets, rest, _rows.check_temperature(temperature)


def _launch(logits, targets, rest, clip, coefs, temperature, ignore_index, grad_dtype, dloss, grad_scale):
    rows, vocab = logits.shape
    old, adv, weights, ref = rest
    dev = logits.device
    loss = old.new_empty(())
    f = old.new_empty((4, rows))  # logp, entropy, kl, and the terms of the sum
    base = f.data_ptr()
    clipped = torch.empty(rows, dtype=torch.bool, device=dev)
    grad = None if grad_dtype is None else _rows.empty_grad(logits, grad_dtype)
    nat.check(
        nat.lib().ferrite_policy_loss(
            nat.stream_ptr(dev), logits.data_ptr(), targets.data_ptr(), old.data_ptr(), adv.data_ptr(), nat.ptr(weights), nat.ptr(ref),
            clip[0], clip[1], coefs[0], coefs[1], temperature, nat.ptr(dloss), grad_scale, loss.data_ptr(), base, base + 4 * rows,
            base + 8 * rows, clipped.data_ptr(), nat.ptr(grad), base + 12 * rows, 4 * rows, rows, vocab, _rows.row_stride(logits), vocab if grad is None else _rows.row_stride(grad), ignore_index,
            nat.dtype_code(logits.dtype), int(targets.dtype == torch.int64), -1 if grad_dtype is None else nat.dtype_code(grad_dtype),
        )
    )
    logp, entropy, kl, _ = f.unbind()
    return PolicyLoss(loss, logp, entropy, kl, clipped), grad


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, rest, clip, coefs, temperature, ignore_index):
        out, _ = _launch(logits, targets, rest, clip, coefs, temperature, ignore_index, None, None, 1.0)
        ctx.save_for_backward(logits, targets, *rest)
        ctx.args = (clip, coefs, temperature, ignore_index)
        ctx.mark_non_differentiable(*out[1:])
        return tuple(out)

    @staticmethod
    @nat.on_tensor_device
    def backward(ctx, g, *_):
        # the row's statistics again and the gradient, in one launch: as much traffic as
        # reading the logits for the gradient alone
        logits, targets, *rest = ctx.saved_tensors
        _, grad = _launch(logits, targets, rest, *ctx.args, logits.dtype, _rows.upstream(g, logits), 1.0)
        return _rows.first_only(grad, logits, g), None, None, None, None, None, None


@nat.on_tensor_device
def policy_loss(logits, targets, old_logprobs, advantages, weights=None, *, ref_logprobs=None, clip_low: float = 0.2, clip_high: float = 0.2,
                kl_coef: float = 0.0, entropy_coef: float = 0.0, temperature: float = 1.0, ignore_index: int = IGNORE_INDEX) -> PolicyLoss:
    """The clipped policy loss of ``logits [rows, vocab]`` (see the top of this file); ``loss`` is
    differentiable in the logits alone, the per-row values are for monitoring.

    targets: int32 or int64, the tokens written.  old_logprobs, advantages, ref_logprobs, weights:
    one value for each row; weights default to ``1 / rows``.  A row of weight zero, or whose target is
    ``ignore_index``, is not read and gives zeros.
    """
    recorded = _rows.differentiable(logits, old_logprobs=old_logprobs, advantages=advantages, weights=weights, ref_logprobs=ref_logprobs)
    targets, rest, temperature = _check(logits, targets, old_logprobs, advantages, weights, ref_logprobs, clip_low, clip_high, temperature, None)
    args = (logits, targets, rest, (float(clip_low), float(clip_high)), (float(kl_coef), float(entropy_coef)), temperature, int(ignore_index))
    if not recorded:
        return _launch(*args, None, None, 1.0)[0]
    return PolicyLoss(*_PolicyLoss.apply(*args))


@nat.on_tensor_device
def policy_loss_and_grad(logits, targets, old_logprobs, advantages, weights=None, *, ref_logprobs=None, clip_low: float = 0.2,
                         clip_high: float = 0.2, kl_coef: float = 0.0, entropy_coef: float = 0.0, temperature: float = 1.0,
                         ignore_index: int = IGNORE_INDEX, grad_scale: float = 1.0, grad_dtype=None,
                         upstream: torch.Tensor | None = None) -> tuple[PolicyLoss, torch.Tensor]:
    """:func:`policy_loss` and ``grad_scale`` times its gradient in the logits, in one pass over
    them; ``grad_dtype`` defaults to the logits' type (f32 logits also give bf16 or f16).  ``upstream``, a scalar
    on the device, multiplies the gradient as well, before it is rounded."""
    grad_dtype = grad_dtype or logits.dtype
    targets, rest, temperature = _check(logits, targets, old_logprobs, advantages, weights, ref_logprobs, clip_low, clip_high, temperature, grad_dtype)
    dloss = None if upstream is None else _rows.upstream(upstream, logits)
    return _launch(logits, targets, rest, (float(clip_low), float(clip_high)), (float(kl_coef), float(entropy_coef)), temperature,
                   int(ignore_index), grad_dtype, dloss, float(grad_scale))


def policy_loss_reference(logits, targets, old_logprobs, advantages, weights=None, *, ref_logprobs=None, clip_low=0.2, clip_high=0.2,
                          kl_coef=0.0, entropy_coef=0.0, temperature=1.0, ignore_index=IGNORE_INDEX) -> PolicyLoss:
    """The same in plain torch f32, differentiable (the definition the kernels are checked against)."""
    from ferrite.kernels.logprobs import token_logprobs_reference

    rows = logits.shape[0]
    w = torch.full((rows,), 1.0 / max(rows, 1), device=logits.device) if weights is None else weights.float()
    live = (w != 0) & (targets != ignore_index)
    logp, h = token_logprobs_reference(logits, torch.where(live, targets, ignore_index), temperature, ignore_index)
    ratio = torch.exp(logp - old_logprobs)
    free, held = ratio * advantages, ratio.clamp(1 - clip_low, 1 + clip_high) * advantages
    d = ref_logprobs - logp if ref_logprobs is not None else torch.zeros_like(logp)
    kl = torch.expm1(d) - d
    per = -torch.minimum(free, held) + kl_coef * kl - entropy_coef * h
    loss = torch.where(live, w * per, 0.0).sum()
    return PolicyLoss(loss, logp.detach(), h.detach(), torch.where(live, kl, 0.0).detach(), (held < free) & live)
