"""RMS norm on MI355X with the residual's addition, with its gradients and with an
8-bit output: the norm that decoder models have in front of each block and of the head.

  rms_norm(x, weight)                     -> y
  rms_norm(x, weight, residual)           -> y, s        s = x + residual
  rms_norm_quantized(x, weight[, residual]) -> q, scales[, s]

Each row is normalised over the last dimension, ``y = s / sqrt(mean(s^2) + eps) *
weight`` with s = x where there is no residual.  s is the stream that goes on past the
block: it has the residual's type, and what is normalised is s as that type holds it, so
that adding and normalising in two steps gives the same.  Statistics and sums are fp32;
y and the gradients are rounded once, the weight's gradient (sums over the rows in a
fixed order: the same bits on every run) to the weight's type.

``rms_norm_quantized`` writes y in 8 bits, e4m3 (``torch.float8_e4m3fn``) or int8, with
fp32 scales per row or per ``group_size`` columns:
  scale = max(largest |y|, 1e-30) / M, M = 448 or 127;  q = round(y / scale) to nearest even
(y, the scale and the quotient in fp32), so that ``q * scale`` stands for y.  It has no
gradient.  A NaN makes its row's (its group's) scale a NaN and an infinity makes it
infinite; their codes stand for nothing.

  * Tensors must live on a HIP device; there is no CPU path.
  * x is bf16, fp16 or fp32 of any shape; the residual has its shape, and its dtype or
    fp32; rows of both may be strided (a last dimension that is not contiguous is
    copied).  weight is [D], of x's dtype or fp32.
  * The results may be changed in place, s only where no backward needs it.  Gradients
    are kernels' results: differentiating them again raises an error.
  * Squares are summed in fp32, as torch's norm does: a row whose sum passes its range
    comes out as 0, and with eps 0 one whose squares vanish has no finite norm.
  * x and a residual of its dtype have one gradient: ``torch.autograd.grad`` returns the
    same tensor for both, as for ``x + residual``; leaves' ``.grad`` are tensors of their
    own.

The reference's norm, without a residual, is triton_kernels.py:2224 (``rmsnorm``); it
quantizes activations in blocks in kernels of their own (fp8_deepseek.py:512-706).
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
import torch.nn as nn

from .. import ops as _ops

__all__ = ["rms_norm", "rms_norm_quantized", "RMSNorm"]

_rms_norm = _ops.rms_norm.default
_rms_norm_quantized = _ops.rms_norm_quantized.default

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_GROUPS = (32, 64, 128, 256)


def _check(x: torch.Tensor, weight: Optional[torch.Tensor], residual: Optional[torch.Tensor], eps: float,
           what: str) -> None:
    if not x.is_cuda:
        raise RuntimeError(f"chronicals_amd {what} runs only on HIP devices: x must be a device tensor (got "
                           f"{x.device})")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError(f"x must be [..., D] with D >= 1, got shape {tuple(x.shape)}")
    if x.dtype not in _FLOATS:
        raise RuntimeError(f"x dtype {x.dtype} not supported (bf16, fp16, fp32)")
    if not (0.0 <= eps < float("inf")):
        raise ValueError(f"eps must be finite and at least 0, got {eps}")
    if weight is not None:
        if weight.dim() != 1 or weight.shape[0] != x.shape[-1]:
            raise RuntimeError(f"weight must be [{x.shape[-1]}], got {tuple(weight.shape)}")
        if weight.device != x.device:
            raise RuntimeError("weight must be on the same device as x")
        if weight.dtype not in (x.dtype, torch.float32):
            raise RuntimeError(f"weight must have x's dtype {x.dtype} or fp32, got {weight.dtype}")
    if residual is not None:
        if residual.shape != x.shape:
            raise RuntimeError(f"residual must have x's shape {tuple(x.shape)}, got {tuple(residual.shape)}")
        if residual.device != x.device:
            raise RuntimeError("residual must be on the same device as x")
        if residual.dtype not in (x.dtype, torch.float32):
            raise RuntimeError(f"residual must have x's dtype {x.dtype} or fp32, got {residual.dtype}")


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """RMS norm of x (or of x + residual) over its last dimension (module docstring); differentiable in x, weight and
    residual.  Returns y, or with a residual (y, x + residual)."""
    _check(x, weight, residual, eps, "rms_norm")
    y, s = _rms_norm(x, weight, residual, eps)
    return y if residual is None else (y, s)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[..., D] as [N, D] with a contiguous last dimension and rows that do not overlap."""
    r = t.detach() if t.requires_grad else t
    if r.dim() != 2:
        r = r.reshape(-1, t.shape[-1])
    if (r.shape[1] > 1 and r.stride(1) != 1) or (r.shape[0] > 1 and r.stride(0) < r.shape[1]):
        r = r.contiguous()
    return r


def rms_norm_quantized(x: torch.Tensor, weight: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                       eps: float = 1e-6, dtype: torch.dtype = torch.float8_e4m3fn,
                       group_size: Optional[int] = None) -> Tuple[torch.Tensor, ...]:
    """RMS norm into 8 bits (module docstring); not differentiable.

    ``dtype`` torch.float8_e4m3fn or torch.int8; ``group_size`` None (a scale per row,
    scales [...]) or 32, 64, 128, 256 (scales [..., ceil(D / group_size)]).  Returns
    (q, scales), with a residual (q, scales, x + residual).
    """
    _check(x, weight, residual, eps, "rms_norm_quantized")
    if dtype not in (torch.float8_e4m3fn, torch.int8):
        raise ValueError(f"dtype must be torch.float8_e4m3fn or torch.int8, got {dtype}")
    if group_size is not None and group_size not in _GROUPS:
        raise ValueError(f"group_size must be None or one of {_GROUPS}, got {group_size}")
    if weight is not None:
        weight = (weight.detach() if weight.requires_grad else weight).contiguous()
    q, scales, s = _rms_norm_quantized(_rows(x), weight, None if residual is None else _rows(residual), eps,
                                       dtype == torch.int8, group_size or 0)
    if x.dim() != 2:
        q, scales = q.view(x.shape), scales.view((*x.shape[:-1], *scales.shape[1:]))
        s = s if residual is None else s.view(x.shape)
    return (q, scales) if residual is None else (q, scales, s)


class RMSNorm(nn.Module):
    """Module form, with the parameter and state dict of torch's nn.RMSNorm over one dimension.

    ``forward(x)`` returns y, ``forward(x, residual)`` (y, x + residual).
    """

    def __init__(self, dim: int, eps: float = 1e-6, elementwise_affine: bool = True, device=None, dtype=None):
        super().__init__()
        self.dim, self.eps = int(dim), eps
        self.weight = nn.Parameter(torch.ones(self.dim, device=device, dtype=dtype)) if elementwise_affine else None

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        if x.dim() < 1 or x.shape[-1] != self.dim:
            raise RuntimeError(f"x must be [..., {self.dim}], got shape {tuple(x.shape)}")
        return rms_norm(x, self.weight, residual, self.eps)

    def extra_repr(self) -> str:
        return f"{self.dim}, eps={self.eps}, elementwise_affine={self.weight is not None}"
