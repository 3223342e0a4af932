"""Log-probabilities (and entropies) of given tokens under logits ``[rows, vocab]``.

The scores that post-training needs next to the training loss: those of the tokens that
were sampled or written, under the model that is trained, the one that sampled them, or a
frozen reference.  One read of the logits (``ferrite_logprobs_fwd``: sums of exponentials
against a base near the row's top, f32 whatever the logits' type); the backward (``ferrite_logprobs_bwd``)
reads them once more and writes the gradient in their type.  No counterpart in the
reference, whose only loss is the mean cross-entropy (src/ferrite/model/gpt.py:147-152).
"""

from __future__ import annotations

import torch

from ferrite import _native as nat
from ferrite.kernels import _rows
from ferrite.kernels._rows import IGNORE_INDEX


def logprobs_forward(logits, targets, temperature: float, ignore_index: int, *, entropy: bool, stats: bool):
    """``(logp, entropy or None, stats or None)`` through ``ferrite_logprobs_fwd``; ``targets`` dense."""
    rows, vocab = logits.shape
    dev = logits.device
    logp = torch.empty(rows, dtype=torch.float32, device=dev)
    h = torch.empty(rows, dtype=torch.float32, device=dev) if entropy else None
    st = torch.empty((rows, 2), dtype=torch.float32, device=dev) if stats else None
    nat.check(
        nat.lib().ferrite_logprobs_fwd(
            nat.stream_ptr(dev), logits.data_ptr(), targets.data_ptr(), logp.data_ptr(), nat.ptr(h), nat.ptr(st),
            rows, vocab, _rows.row_stride(logits), ignore_index, temperature, nat.dtype_code(logits.dtype),
            int(targets.dtype == torch.int64),
        )
    )
    return logp, h, st


def logprobs_backward(logits, targets, stats, entropy, dlogp, dentropy, dloss, scale: float, temperature: float, ignore_index: int, out_dtype):
    """The gradient of ``sum(dlogp * logp + dentropy * H) * dloss * scale`` through ``ferrite_logprobs_bwd``."""
    rows, vocab = logits.shape
    out = _rows.empty_grad(logits, out_dtype)
    nat.check(
        nat.lib().ferrite_logprobs_bwd(
            nat.stream_ptr(logits.device), logits.data_ptr(), targets.data_ptr(), stats.data_ptr(), nat.ptr(entropy), nat.ptr(dlogp),
            nat.ptr(dentropy), nat.ptr(dloss), scale, out.data_ptr(), rows, vocab, _rows.row_stride(logits), _rows.row_stride(out), ignore_index,
            temperature, nat.dtype_code(logits.dtype), int(targets.dtype == torch.int64), nat.dtype_code(out_dtype),
        )
    )
    return out


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, temperature, entropy, ignore_index):
        logp, h, stats = logprobs_forward(logits, targets, temperature, ignore_index, entropy=entropy, stats=True)
        ctx.save_for_backward(logits, targets, stats, h)
        ctx.temperature, ctx.ignore_index = temperature, ignore_index
        return (logp, h) if entropy else logp

    @staticmethod
    @nat.on_tensor_device
    def backward(ctx, dlogp, dentropy=None):
        logits, targets, stats, h = ctx.saved_tensors
        rows = logits.shape[0]
        grad = logprobs_backward(
            logits, targets, stats, h, _rows.per_row(dlogp, rows, "dlogp"), _rows.per_row(dentropy, rows, "dentropy"), None, 1.0,
            ctx.temperature, ctx.ignore_index, logits.dtype)
        return _rows.first_only(grad, logits, dlogp, dentropy), None, None, None, None


@nat.on_tensor_device
def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *, temperature: float = 1.0, entropy: bool = False,
                   ignore_index: int = IGNORE_INDEX):
    """``log softmax(logits / temperature)`` at ``targets``: f32 ``[rows]``; with ``entropy`` the pair
    ``(logp, H)``, ``H`` the entropy of each row's distribution.  Differentiable in the logits.

    logits: ``[rows, vocab]`` f32, bf16 or f16, unit column stride, any row stride.  targets: int32 or
    int64, one for each row; a row whose target is ``ignore_index`` is not read and gives zeros; another
    target outside ``[0, vocab)`` gives NaN.
    """
    rows, _ = _rows.check_logits(logits)
    targets, _ = _rows.check_targets(targets, rows)
    temperature = _rows.check_temperature(temperature)
    _rows.same_device(logits, targets)
    if not _rows.differentiable(logits):
        logp, h, _ = logprobs_forward(logits, targets, temperature, int(ignore_index), entropy=entropy, stats=False)
        return (logp, h) if entropy else logp
    return _TokenLogprobs.apply(logits, targets, temperature, bool(entropy), int(ignore_index))


def token_logprobs_reference(logits, targets, temperature: float = 1.0, ignore_index: int = IGNORE_INDEX):
    """``(logp, H)`` in plain torch, f32 (the definition the kernels are checked against)."""
    lp = torch.log_softmax(logits.float() / temperature, dim=-1)
    live = targets != ignore_index
    logp = lp.gather(1, torch.where(live, targets, 0).long()[:, None])[:, 0]
    p = lp.exp()
    h = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    return torch.where(live, logp, 0.0), torch.where(live, h, 0.0)
