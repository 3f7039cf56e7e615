"""Distillation from a teacher's top logits, on MI355X.

A teacher's answer for a token is kept as its K largest logits and their columns
(``top_logits``).  The student is trained towards softmax(t / T) over those K, in
the two forms that the cross-entropy has here:

  distillation_loss, DistillationLoss
      over student logits that exist (as ``chunked_cross_entropy_loss``): the
      forward streams them once, the backward again, writing the gradient.
  linear_distillation_loss, LinearDistillationLoss
      from hidden states and the head's weight (as ``cut_cross_entropy``): the
      student's N x V logits are never stored.

Per row, with q = softmax(t / T) over the row's usable entries (t_k, i_k):

  distill_weight * T^2 * sum_k q_k * (log q_k - log softmax(x / T)[i_k])
    + ce_weight * (logsumexp(x) - x[label])

so with ``ce_weight`` the labels' loss comes from the same passes.

  * An entry whose index is outside [0, V) (use -1 as padding) or whose logit is
    -inf takes no part, whatever else it holds; a row left without any has no
    distillation term.  Entries that share an index add up there.
  * ``labels``: a row labelled ``ignore_index`` gives no loss and a zero gradient,
    whatever its logits hold; its hidden states have to be finite in the linear
    form, whose products run over them with zero coefficients.
    A label outside [0, V) that is not ``ignore_index`` has no target logit.
    Without labels (``ce_weight`` is 0 then) a row counts if it has a usable entry.
  * 'mean' divides by the number of rows that count, at least 1; 'sum' adds them;
    'none' returns one value per row, in the shape of the rows.
  * K is at most 256, the temperature in [0.01, 1000].
  * Losses are fp32.  Sums are added in a fixed order: the same bits on every run.
  * Tensors must live on a HIP device; there is no CPU path.  The teacher's
    tensors get no gradient.  Losses may be changed in place.  Differentiating a
    gradient again raises an error, and so do function transforms
    (``torch.func``, forward mode).
  * ``linear_distillation_loss`` computes in bf16 with fp32 accumulation (fp16 and
    fp32 operands are rounded to bf16 at the boundary) and rounds the gradient of
    the logits to bf16 once, as ``cut_cross_entropy`` does, in units that hold the
    label's share of it exactly; gradients come back in the input dtypes.

The reference has no distillation; the argument order follows its losses.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn

from .. import _lib
from .. import ops as _ops
from .cut_cross_entropy import _reduction_code, get_optimal_chunk_size

__all__ = [
    "top_logits",
    "distillation_loss",
    "DistillationLoss",
    "linear_distillation_loss",
    "LinearDistillationLoss",
]

_top_logits = _ops.top_logits.default
_distill_logits = _ops.distill_logits.default
_distill_linear = _ops.distill_linear.default

MAX_ENTRIES = _lib.CCE_MAX_TEACHER_ENTRIES
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_INTS = (torch.int64, torch.int32)


def _logit_rows(logits: torch.Tensor) -> torch.Tensor:
    """[..., V] as [N, V] with a contiguous last dimension and rows that do not overlap."""
    x = logits.reshape(-1, logits.shape[-1])
    if (x.shape[1] > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    return x


def _check_student(x: torch.Tensor, name: str, what: str) -> None:
    if not x.is_cuda:
        raise RuntimeError(f"chronicals_amd {what} runs only on HIP devices: {name} must be a device tensor (got "
                           f"{x.device})")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError(f"{name} must be [..., D] with D >= 1, got shape {tuple(x.shape)}")
    if x.dtype not in _FLOATS:
        raise RuntimeError(f"{name} dtype {x.dtype} not supported (bf16, fp16, fp32)")


def _teacher_rows(student: torch.Tensor, teacher_logits: torch.Tensor, teacher_indices: torch.Tensor,
                  labels: Optional[torch.Tensor], temperature: float, ce_weight: float):
    """The teacher's tensors as contiguous [N, K] and the labels as [N], for a student of shape [..., D]."""
    shape = teacher_logits.shape
    if teacher_logits.dim() < 1 or shape[:-1] != student.shape[:-1]:
        raise RuntimeError(f"teacher_logits must be {[*student.shape[:-1], 'K']}, got {tuple(shape)}")
    if teacher_indices.shape != shape:
        raise RuntimeError(f"teacher_indices must have the shape {tuple(shape)} of teacher_logits, got "
                           f"{tuple(teacher_indices.shape)}")
    if not 1 <= shape[-1] <= MAX_ENTRIES:
        raise RuntimeError(f"a teacher has 1 to {MAX_ENTRIES} entries per row, got {shape[-1]}")
    if teacher_logits.dtype not in _FLOATS:
        raise RuntimeError(f"teacher_logits dtype {teacher_logits.dtype} not supported (bf16, fp16, fp32)")
    if teacher_indices.dtype not in _INTS:
        raise RuntimeError(f"teacher_indices must be int64 or int32, got {teacher_indices.dtype}")
    if teacher_logits.device != student.device or teacher_indices.device != student.device:
        raise RuntimeError("teacher_logits and teacher_indices must be on the student's device")
    if not 1e-2 <= temperature <= 1e3:
        raise ValueError(f"temperature must be in [0.01, 1000], got {temperature}")
    n = shape[:-1].numel()
    if labels is None:
        if ce_weight != 0.0:
            raise ValueError("ce_weight needs labels")
    else:
        if labels.dtype not in _INTS:
            raise RuntimeError(f"labels must be int64 or int32, got {labels.dtype}")
        if labels.numel() != n:
            raise RuntimeError(f"labels has {labels.numel()} elements but the student has {n} rows")
        if labels.device != student.device:
            raise RuntimeError("labels must be on the student's device")
        labels = labels.reshape(-1).contiguous()
    return (teacher_logits.detach().reshape(n, shape[-1]).contiguous(),
            teacher_indices.reshape(n, shape[-1]).contiguous(), labels)


def top_logits(logits: torch.Tensor, k: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """The k largest of each row of [..., V] logits, largest first, and their indices (int64): [..., k] each.

    Among equal values the lower index comes first; NaN is larger than any
    number and -0 equals +0.  1 <= k <= min(V, 256).  Not differentiable: a
    teacher's answer.
    """
    _check_student(logits, "logits", "top_logits")
    V = logits.shape[-1]
    if not 1 <= k <= min(V, MAX_ENTRIES):
        raise ValueError(f"k must be in [1, min({MAX_ENTRIES}, V = {V})], got {k}")
    values, indices = _top_logits(_logit_rows(logits.detach()), int(k))
    shape = (*logits.shape[:-1], k)
    return values.view(shape), indices.view(shape)


def distillation_loss(
    logits: torch.Tensor,
    teacher_logits: torch.Tensor,
    teacher_indices: torch.Tensor,
    labels: Optional[torch.Tensor] = None,
    temperature: float = 1.0,
    distill_weight: float = 1.0,
    ce_weight: float = 0.0,
    ignore_index: int = -100,
    reduction: str = "mean",
) -> torch.Tensor:
    """Distillation loss over student logits [..., V] that exist (module docstring); differentiable in ``logits``.

    teacher_logits and teacher_indices [..., K]; labels [...] or None.
    """
    red = _reduction_code(reduction)
    _check_student(logits, "logits", "distillation_loss")
    t, index, lab = _teacher_rows(logits, teacher_logits, teacher_indices, labels, temperature, ce_weight)
    loss = _distill_logits(logits, t, index, lab, temperature, distill_weight, ce_weight, ignore_index, red)
    return loss.view(logits.shape[:-1]) if red == _lib.CCE_REDUCTION_NONE else loss


class DistillationLoss(nn.Module):
    """Module form of distillation_loss."""

    def __init__(self, temperature: float = 1.0, distill_weight: float = 1.0, ce_weight: float = 0.0,
                 ignore_index: int = -100, reduction: str = "mean"):
        super().__init__()
        _reduction_code(reduction)
        self.temperature = temperature
        self.distill_weight = distill_weight
        self.ce_weight = ce_weight
        self.ignore_index = ignore_index
        self.reduction = reduction

    def forward(self, logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_indices: torch.Tensor,
                labels: Optional[torch.Tensor] = None) -> torch.Tensor:
        return distillation_loss(logits, teacher_logits, teacher_indices, labels, self.temperature,
                                 self.distill_weight, self.ce_weight, self.ignore_index, self.reduction)

    def extra_repr(self) -> str:
        return (f"temperature={self.temperature}, distill_weight={self.distill_weight}, "
                f"ce_weight={self.ce_weight}, ignore_index={self.ignore_index}, reduction={self.reduction!r}")


def linear_distillation_loss(
    hidden: torch.Tensor,
    weight: torch.Tensor,
    teacher_logits: torch.Tensor,
    teacher_indices: torch.Tensor,
    labels: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    chunk_size: int = 8192,
    temperature: float = 1.0,
    distill_weight: float = 1.0,
    ce_weight: float = 0.0,
    ignore_index: int = -100,
    reduction: str = "mean",
) -> torch.Tensor:
    """Fused lm_head projection + distillation loss without materialising logits (module docstring).

    hidden [..., d], weight [V, d], bias [V] or None, teacher_logits and
    teacher_indices [..., K], labels [...] or None; differentiable in hidden,
    weight and bias.  d is a multiple of 8.  ``chunk_size`` bounds the backward's
    vocabulary band, as in ``cut_cross_entropy``.
    """
    red = _reduction_code(reduction)
    _check_student(hidden, "hidden", "linear_distillation_loss")
    if weight.dim() != 2:
        raise RuntimeError(f"weight must be [vocab_size, hidden_dim], got shape {tuple(weight.shape)}")
    if weight.device != hidden.device:
        raise RuntimeError("hidden and weight must be on the same device")
    if weight.dtype not in _FLOATS:
        raise RuntimeError(f"weight dtype {weight.dtype} not supported (bf16, fp16, fp32)")
    if hidden.shape[-1] != weight.shape[1]:
        raise RuntimeError(f"hidden last dim {hidden.shape[-1]} does not match weight hidden_dim {weight.shape[1]}")
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != weight.shape[0]:
            raise RuntimeError(f"bias must be [vocab_size={weight.shape[0]}], got {tuple(bias.shape)}")
        if bias.device != hidden.device:
            raise RuntimeError("bias must be on the same device as hidden")
    t, index, lab = _teacher_rows(hidden, teacher_logits, teacher_indices, labels, temperature, ce_weight)
    loss = _distill_linear(hidden, weight, bias, t, index, lab, chunk_size, temperature, distill_weight, ce_weight,
                           ignore_index, red)
    return loss.view(hidden.shape[:-1]) if red == _lib.CCE_REDUCTION_NONE else loss


class LinearDistillationLoss(nn.Module):
    """Module form of linear_distillation_loss; ``chunk_size=None`` picks ``get_optimal_chunk_size`` per call, as
    CutCrossEntropyLoss does."""

    def __init__(self, chunk_size: Optional[int] = None, temperature: float = 1.0, distill_weight: float = 1.0,
                 ce_weight: float = 0.0, ignore_index: int = -100, reduction: str = "mean"):
        super().__init__()
        _reduction_code(reduction)
        self.chunk_size = chunk_size
        self.temperature = temperature
        self.distill_weight = distill_weight
        self.ce_weight = ce_weight
        self.ignore_index = ignore_index
        self.reduction = reduction

    def forward(self, hidden: torch.Tensor, weight: torch.Tensor, teacher_logits: torch.Tensor,
                teacher_indices: torch.Tensor, labels: Optional[torch.Tensor] = None,
                bias: Optional[torch.Tensor] = None) -> torch.Tensor:
        chunk = self.chunk_size
        if chunk is None:
            chunk = get_optimal_chunk_size(weight.shape[0], weight.shape[1])
        return linear_distillation_loss(hidden, weight, teacher_logits, teacher_indices, labels, bias, chunk,
                                        self.temperature, self.distill_weight, self.ce_weight, self.ignore_index,
                                        self.reduction)

    def extra_repr(self) -> str:
        return (f"chunk_size={self.chunk_size}, temperature={self.temperature}, "
                f"distill_weight={self.distill_weight}, ce_weight={self.ce_weight}, "
                f"ignore_index={self.ignore_index}, reduction={self.reduction!r}")
