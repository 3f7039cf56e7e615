"""Layer norm on MI355X, with its gradients: the norm in front of the head.

``layer_norm(x, weight, bias, eps)`` normalises each row over the last dimension,
``(x - mean) / sqrt(var + eps) * weight + bias``, as torch's functional of that
name does.  Statistics and sums are fp32 whatever the input's type; the output
and the input's gradient are rounded once to the input's type, the parameters'
gradients (sums over the rows in a fixed order: the same bits on every run) to
the parameters'.

  * Tensors must live on a HIP device; there is no CPU path.
  * x is bf16, fp16 or fp32 of any shape; rows may be strided (a last dimension
    that is not contiguous is copied).  weight and bias are [D], either or both,
    of x's dtype or fp32, both alike.
  * The output may be changed in place.  Its gradients are kernels' results:
    differentiating them again raises an error.

The reference has no layer norm of its own; the models that it fine-tunes bring
torch's.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from .. import ops as _ops

__all__ = ["layer_norm", "LayerNorm"]

_layer_norm = _ops.layer_norm.default


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm of x over its last dimension; differentiable in x, weight and bias."""
    if not x.is_cuda:
        raise RuntimeError(f"chronicals_amd layer_norm runs only on HIP devices: x must be a device tensor (got "
                           f"{x.device})")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError(f"x must be [..., D] with D >= 1, got shape {tuple(x.shape)}")
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise RuntimeError(f"x dtype {x.dtype} not supported (bf16, fp16, fp32)")
    if not (0.0 <= eps < float("inf")):
        raise ValueError(f"eps must be finite and at least 0, got {eps}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.dim() != 1 or p.shape[0] != x.shape[-1]:
            raise RuntimeError(f"{name} must be [{x.shape[-1]}], got {tuple(p.shape)}")
        if p.device != x.device:
            raise RuntimeError(f"{name} must be on the same device as x")
        if p.dtype not in (x.dtype, torch.float32):
            raise RuntimeError(f"{name} must have x's dtype {x.dtype} or fp32, got {p.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError(f"weight and bias must have the same dtype, got {weight.dtype} and {bias.dtype}")
    return _layer_norm(x, weight, bias, eps)


class LayerNorm(nn.Module):
    """Module form, with the parameters and state dict of torch's nn.LayerNorm over one dimension."""

    def __init__(self, dim: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, device=None,
                 dtype=None):
        super().__init__()
        self.dim, self.eps = int(dim), eps
        self.weight = nn.Parameter(torch.ones(self.dim, device=device, dtype=dtype)) if elementwise_affine else None
        self.bias = (nn.Parameter(torch.zeros(self.dim, device=device, dtype=dtype)) if elementwise_affine and bias
                     else None)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dim() < 1 or x.shape[-1] != self.dim:
            raise RuntimeError(f"x must be [..., {self.dim}], got shape {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self) -> str:
        return f"{self.dim}, eps={self.eps}, elementwise_affine={self.weight is not None}"
