"""The preference loss of pairs of sequences, over the packed logits ``[rows, vocab]`` of all of them.

``offsets`` cut the rows into ``2 pairs`` sequences, ``2p`` the chosen and ``2p + 1`` the rejected one
of pair ``p``.  With ``logp_r`` the log-probability of the token written at row ``r``::

    d_j  = sum over sequence j of (logp_r - ref_logprobs_r)     (``average``: divided by its live rows)
    h    = d_2p - d_2p+1
    loss = mean over pairs of  -(1 - e) log sigmoid(beta h) - e log sigmoid(-beta h)    "sigmoid", e = label_smoothing
                               (h - 1 / (2 beta))^2                                     "squared"
                               max(0, 1 - beta h)                                       "hinge"

Three launches: the rows' log-probabilities (one read of the logits), the pairs (sums in f64, a
fixed order), and the gradient (a second read -- no row's coefficient is known before its
pair's last row has been scored -- and the write).  No counterpart in the reference, whose only
loss is the mean cross-entropy (src/ferrite/model/gpt.py:147-152).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ferrite import _native as nat
from ferrite.kernels import _rows
from ferrite.kernels._rows import IGNORE_INDEX
from ferrite.kernels.logprobs import logprobs_backward

KINDS = ("sigmoid", "squared", "hinge")


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor  # f32 scalar
    margins: torch.Tensor  # f32 [pairs]: beta h
    logprobs: torch.Tensor  # f32 [rows]; zeros for masked rows


def _check(logits, targets, ref_logprobs, offsets, beta, kind, label_smoothing, temperature, grad_dtype):
    rows, _ = _rows.check_logits(logits, grad_dtype)
    targets, _ = _rows.check_targets(targets, rows)
    if offsets.ndim != 1 or offsets.numel() < 3 or offsets.numel() % 2 == 0:
        raise ValueError(f"offsets must hold 2 * pairs + 1 row numbers, got shape {tuple(offsets.shape)}")
    if offsets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"offsets must be int32 or int64, got {offsets.dtype}")
    if kind not in KINDS:
        raise ValueError(f"kind must be one of {KINDS}, got {kind!r}")
    if not 0.0 <= label_smoothing < 0.5:
        raise ValueError(f"label_smoothing must lie in [0, 0.5), got {label_smoothing}")
    if not 0.0 < float(beta) < float("inf"):
        raise ValueError(f"beta must be positive and finite, got {beta}")
    ref = _rows.per_row(ref_logprobs, rows, "ref_logprobs")
    _rows.same_device(logits, targets, ref, offsets)
    if offsets.dtype != torch.int64 or not offsets.is_contiguous():
        offsets = offsets.to(torch.int64).contiguous()
    return targets, ref, offsets, _rows.check_temperature(temperature)


def _launch(logits, targets, ref, offsets, beta, kind, label_smoothing, average, temperature, ignore_index, keep, grad_dtype, grad_scale):
    """``(PreferenceLoss, stats, coef, gradient)``; ``keep`` the rows' statistics and coefficients for a backward."""
    rows, vocab = logits.shape
    pairs, dev = offsets.numel() // 2, logits.device
    keep = keep or grad_dtype is not None
    loss = ref.new_empty(())
    per_pair = ref.new_empty((2, pairs))  # margins and the terms of the mean
    logp = ref.new_empty(rows)
    stats = ref.new_empty((rows, 2)) if keep else None
    coef = ref.new_empty(rows) if keep else None
    grad = None if grad_dtype is None else _rows.empty_grad(logits, grad_dtype)
    base = per_pair.data_ptr()
    nat.check(
        nat.lib().ferrite_preference_loss(
            nat.stream_ptr(dev), logits.data_ptr(), targets.data_ptr(), ref.data_ptr(), offsets.data_ptr(), beta, label_smoothing,
            KINDS.index(kind), int(average), temperature, grad_scale, loss.data_ptr(), base, logp.data_ptr(), nat.ptr(stats), nat.ptr(coef),
            nat.ptr(grad), base + 4 * pairs, 4 * pairs, rows, pairs, vocab, _rows.row_stride(logits),
            vocab if grad is None else _rows.row_stride(grad), ignore_index, nat.dtype_code(logits.dtype), int(targets.dtype == torch.int64),
            -1 if grad is None else nat.dtype_code(grad_dtype),
        )
    )
    return PreferenceLoss(loss, per_pair.unbind()[0], logp), stats, coef, grad


class _Preference(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, ref, offsets, beta, kind, label_smoothing, average, temperature, ignore_index):
        out, stats, coef, _ = _launch(logits, targets, ref, offsets, beta, kind, label_smoothing, average, temperature, ignore_index, True, None, 1.0)
        ctx.save_for_backward(logits, targets, stats, coef)
        ctx.temperature, ctx.ignore_index = temperature, ignore_index
        ctx.mark_non_differentiable(*out[1:])
        return tuple(out)

    @staticmethod
    @nat.on_tensor_device
    def backward(ctx, g, *_):
        logits, targets, stats, coef = ctx.saved_tensors
        grad = logprobs_backward(logits, targets, stats, None, coef, None, _rows.upstream(g, logits), 1.0, ctx.temperature, ctx.ignore_index, logits.dtype)
        return (_rows.first_only(grad, logits, g), *([None] * 9))


@nat.on_tensor_device
def preference_loss(logits, targets, ref_logprobs, offsets, *, beta: float = 0.1, kind: str = "sigmoid", label_smoothing: float = 0.0,
                    average: bool = False, temperature: float = 1.0, ignore_index: int = IGNORE_INDEX) -> PreferenceLoss:
    """The preference loss of the packed ``logits [rows, vocab]`` (see the top of this file); ``loss`` is
    differentiable in the logits alone.

    targets: int32 or int64; rows whose target is ``ignore_index`` (prompts, padding) are not read and
    count in no sequence.  ref_logprobs: the reference model's, one for each row.  offsets: int32 or
    int64 ``[2 pairs + 1]`` on the device, non-decreasing row numbers; rows outside every sequence get
    no gradient.  label_smoothing is the sigmoid loss's; the others do not use it.
    """
    recorded = _rows.differentiable(logits, ref_logprobs=ref_logprobs)
    targets, ref, offsets, temperature = _check(logits, targets, ref_logprobs, offsets, beta, kind, label_smoothing, temperature, None)
    args = (logits, targets, ref, offsets, float(beta), kind, float(label_smoothing), bool(average), temperature, int(ignore_index))
    if not recorded:
        return _launch(*args, False, None, 1.0)[0]
    return PreferenceLoss(*_Preference.apply(*args))


@nat.on_tensor_device
def preference_loss_and_grad(logits, targets, ref_logprobs, offsets, *, beta: float = 0.1, kind: str = "sigmoid", label_smoothing: float = 0.0,
                             average: bool = False, temperature: float = 1.0, ignore_index: int = IGNORE_INDEX, grad_scale: float = 1.0,
                             grad_dtype=None, upstream: torch.Tensor | None = None) -> tuple[PreferenceLoss, torch.Tensor]:
    """:func:`preference_loss` and ``grad_scale`` times its gradient in the logits; ``grad_dtype``
    defaults to the logits' type (f32 logits also give bf16 or f16).  ``upstream``, a scalar on the device, multiplies
    the gradient as well, before it is rounded."""
    grad_dtype = grad_dtype or logits.dtype
    targets, ref, offsets, temperature = _check(logits, targets, ref_logprobs, offsets, beta, kind, label_smoothing, temperature, grad_dtype)
    dloss = None if upstream is None else _rows.upstream(upstream, logits)
    out, stats, coef, grad = _launch(logits, targets, ref, offsets, float(beta), kind, float(label_smoothing), average, temperature, int(ignore_index),
                                     True, grad_dtype if dloss is None else None, float(grad_scale))
    if dloss is not None:
        grad = logprobs_backward(logits, targets, stats, None, coef, None, dloss, float(grad_scale), temperature, int(ignore_index), grad_dtype)
    return out, grad


def preference_loss_reference(logits, targets, ref_logprobs, offsets, *, beta=0.1, kind="sigmoid", label_smoothing=0.0, average=False,
                              temperature=1.0, ignore_index=IGNORE_INDEX) -> PreferenceLoss:
    """The same in plain torch f32, differentiable (the definition the kernels are checked against)."""
    from ferrite.kernels.logprobs import token_logprobs_reference

    logp, _ = token_logprobs_reference(logits, targets, temperature, ignore_index)
    live = targets != ignore_index
    ratio = torch.where(live, logp - ref_logprobs, 0.0)
    at = torch.arange(logits.shape[0], device=logits.device)
    inside = (at >= offsets[:-1, None]) & (at < offsets[1:, None]) & live
    d = torch.where(inside, ratio, 0.0).sum(1)
    if average:
        d = d / inside.sum(1).clamp_min(1)
    h = d[0::2] - d[1::2]
    if kind == "sigmoid":
        ls = torch.nn.functional.logsigmoid
        per = -(1 - label_smoothing) * ls(beta * h) - label_smoothing * ls(-beta * h)
    elif kind == "squared":
        per = (h - 0.5 / beta) ** 2
    else:
        per = torch.relu(1 - beta * h)
    return PreferenceLoss(per.mean(), (beta * h).detach(), logp.detach())
