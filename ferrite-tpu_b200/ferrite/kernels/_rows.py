"""Argument checks and buffers that the losses over logits ``[rows, vocab]`` share
(:mod:`ferrite.kernels.logprobs`, ``policy_loss``, ``preference_loss``, ``distillation``).

A call on a few rows takes less time on the GPU than its checks in Python, so these look at each tensor
once and leave a tensor that is already as the kernels want it alone."""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from ferrite import _native as nat

IGNORE_INDEX = -100


def check_logits(logits: torch.Tensor, grad_dtype=None) -> tuple[int, int]:
    """(rows, vocab) of a 2-D tensor of f32, bf16 or f16 with unit column stride, rows apart by at
    least ``vocab`` elements; ``grad_dtype`` is its own type, or a 16-bit one for f32 logits."""
    if logits.dim() != 2:
        raise ValueError(f"logits must be [rows, vocab], got {tuple(logits.shape)}")
    code = nat.dtype_code(logits.dtype)
    rows, vocab = logits.shape
    if vocab < 1:
        raise ValueError("logits need at least one column")
    if not logits.is_contiguous():
        between, within = logits.stride()
        if (within != 1 and vocab > 1) or (rows > 1 and between < vocab):
            raise ValueError(f"logits must have unit column stride and rows that do not overlap, got strides {logits.stride()}")
    if grad_dtype is not None and grad_dtype != logits.dtype and not (code == nat.F32 and grad_dtype in (torch.bfloat16, torch.float16)):
        raise TypeError(f"gradient of type {grad_dtype} for logits of type {logits.dtype}: expected the logits' own, or 16-bit for float32")
    return rows, vocab


def row_stride(logits: torch.Tensor) -> int:
    """The stride between rows in elements (of a single row: its length)."""
    rows, vocab = logits.shape
    return max(logits.stride(0), vocab) if rows > 1 else vocab


def empty_grad(logits: torch.Tensor, dtype) -> torch.Tensor:
    """An uninitialised ``[rows, vocab]`` gradient, its rows apart and aligned as the logits' are (so
    that a kernel can move both in the same vectors); dense where the logits' rows lie far apart."""
    lead = logits.data_ptr() % 16 // logits.element_size()
    if not lead and logits.is_contiguous():
        return torch.empty_like(logits) if dtype == logits.dtype else torch.empty_like(logits, dtype=dtype)
    rows, vocab = logits.shape
    ld = row_stride(logits)
    if ld > vocab + max(64, vocab // 16):
        ld = vocab
    if ld == vocab and not lead:
        return torch.empty((rows, vocab), dtype=dtype, device=logits.device)
    return torch.empty(rows * ld + lead, dtype=dtype, device=logits.device).as_strided((rows, vocab), (ld, 1), lead)


def check_targets(targets: torch.Tensor, rows: int) -> tuple[torch.Tensor, int]:
    """(targets as one dense row, their type's code): int32 or int64, one for each row of logits."""
    code = 1 if targets.dtype == torch.int64 else 0
    if not code and targets.dtype != torch.int32:
        raise TypeError(f"targets must be int32 or int64, got {targets.dtype}")
    if targets.numel() != rows:
        raise ValueError(f"{targets.numel()} targets for {rows} rows")
    return targets if targets.is_contiguous() else targets.reshape(-1).contiguous(), code


def per_row(t: torch.Tensor | None, rows: int, name: str) -> torch.Tensor | None:
    """A dense f32 tensor of one value for each row."""
    if t is None:
        return None
    if t.numel() != rows:
        raise ValueError(f"{name}: {t.numel()} values for {rows} rows")
    if t.dtype == torch.float32 and t.is_contiguous():
        return t
    if not t.is_floating_point():
        raise TypeError(f"{name} must be floating point, got {t.dtype}")
    return t.detach().reshape(-1).to(torch.float32).contiguous()


def check_temperature(temperature: float) -> float:
    temperature = float(temperature)
    if not (temperature > 0.0 and math.isfinite(temperature)):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    return temperature


def upstream(g: torch.Tensor, logits: torch.Tensor) -> torch.Tensor:
    """The gradient of a scalar loss as a dense f32 scalar on the logits' device."""
    if g.numel() != 1 or not g.is_floating_point():
        raise ValueError(f"the upstream gradient must be one floating-point number, got {g.dtype} of shape {tuple(g.shape)}")
    same_device(logits, g)
    return g.detach().reshape(()).to(torch.float32).contiguous()


def same_device(logits: torch.Tensor, *others: torch.Tensor | None) -> None:
    """Refuses tensors that are not all on one GPU."""
    if not logits.is_cuda:
        nat.require_cuda(logits)
    index = logits.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            nat.require_cuda(t)
            raise ValueError(f"tensors on {logits.device} and {t.device}: expected one device")


def recorded(*tensors: torch.Tensor) -> bool:
    """Whether autograd is to see a call on these: for a gradient, or for a forward-mode tangent (which its
    function then refuses)."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        return True
    return any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def differentiable(logits: torch.Tensor, **others: torch.Tensor | None) -> bool:
    """Whether a call on these logits is to be recorded.  The losses have a gradient in the logits only: where it
    is recorded, another argument that asks for one is refused."""
    if not recorded(logits):
        return False
    for name, t in others.items():
        if t is not None and t.requires_grad:
            raise ValueError(f"{name} requires a gradient, but the loss is differentiable in the logits only: pass it detached")
    return True


class _FirstOnly(torch.autograd.Function):
    @staticmethod
    def forward(ctx, grad, *sources):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("the losses over logits have no second derivative")


def first_only(grad: torch.Tensor | None, *sources: torch.Tensor | None) -> torch.Tensor | None:
    """A backward's result.  Where it is itself recorded (``create_graph``), what it depends on is named by ``sources``, so
    that a second backward raises instead of passing it by as a constant."""
    return grad if grad is None or not torch.is_grad_enabled() else _FirstOnly.apply(grad, *sources)
