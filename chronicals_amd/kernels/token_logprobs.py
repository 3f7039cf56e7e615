"""Log-probabilities of given tokens, entropies and top alternatives, on MI355X.

What policy and preference training and scoring take from a model's answer, in the
two forms that the cross-entropy has here:

  token_logprobs
      over logits that exist (as ``chunked_cross_entropy_loss``): the forward streams
      them once, the backward again, writing the gradient.
  linear_token_logprobs
      from hidden states and the head's weight (as ``cut_cross_entropy``): without
      alternatives the N x V logits are never stored, with them a block of rows'
      at a time.

Per row, with z = x / temperature and p = softmax(z):

  logprobs = z[token] - logsumexp(z)          entropy = -sum_v p_v log p_v
  top_logprobs, top_indices: z - logsumexp(z) at the ``top_k`` largest logits,
  largest first, among equal ones the lower column first, as ``top_logits`` orders them

  * Both results are fp32, in the shape of the rows, and differentiable; the
    alternatives are not.  Either may be left without a gradient.
  * A row whose token is ``ignore_index`` gives 0 for both, alternatives of 0 at
    column -1, and a zero gradient, whatever its logits hold; its hidden states have
    to be finite in the linear form, whose products run over them with zero
    coefficients.
  * A token outside [0, V) that is not ``ignore_index`` has no log-probability: 0,
    without a gradient.  The row's entropy and alternatives are as any other's.
  * Logits of -inf have no probability and take no part; where all of a row's are,
    its log-probabilities are -inf, its entropy 0 and its gradient 0.  In the linear form
    a row whose logits over the temperature are all below -1e30 log(2) counts as such a
    one (a bias of fp32's lowest value in every column); beside others such a column is
    one of probability 0, whose log-probability is what fp32 holds of it.
  * top_k is at most min(V, 256), the temperature in [0.01, 1000].
  * Sums are added in a fixed order: the same bits on every run.
  * Tensors must live on a HIP device; there is no CPU path.  Results may be changed in
    place.  Differentiating a gradient again raises an error, and so do function
    transforms (``torch.func``, forward mode).
  * ``linear_token_logprobs`` computes in bf16 with fp32 accumulation (fp16 and fp32
    operands are rounded to bf16 at the boundary) and rounds the gradient of the logits
    to bf16 once, in units that hold the largest token's share of it exactly; gradients
    come back in the input dtypes.  The token's logit is a dot product beside the one of
    the sums: the order of the additions, some 2^-24 of a logit's terms, is left even in
    rows that are sure of their token (3e-6 of -0.3 under logits of 15).

For a token in [0, V) ``-logprobs`` at temperature 1 is the loss of ``cut_cross_entropy``
with reduction 'none'.  Logits that are NaN or +inf make their row's results NaN.
The reference has no counterpart; the argument order follows its losses.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .. import ops as _ops
from .distillation import _FLOATS, _INTS, MAX_ENTRIES, _check_student

__all__ = ["TokenLogprobs", "token_logprobs", "linear_token_logprobs"]

_token_logprobs = _ops.token_logprobs.default
_linear_token_logprobs = _ops.linear_token_logprobs.default


class TokenLogprobs(NamedTuple):
    """Results of N rows in their shape; the alternatives [..., top_k], None without any."""
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: Optional[torch.Tensor]
    top_indices: Optional[torch.Tensor]


def _check(x: torch.Tensor, tokens: torch.Tensor, V: int, temperature: float, top_k: int) -> torch.Tensor:
    """The tokens as contiguous [N], for x [..., D]."""
    if tokens.dtype not in _INTS:
        raise RuntimeError(f"tokens must be int64 or int32, got {tokens.dtype}")
    if tokens.shape != x.shape[:-1]:
        raise RuntimeError(f"tokens must be {list(x.shape[:-1])}, got {tuple(tokens.shape)}")
    if tokens.device != x.device:
        raise RuntimeError("tokens must be on the device of the logits or hidden states")
    if not 1e-2 <= temperature <= 1e3:
        raise ValueError(f"temperature must be in [0.01, 1000], got {temperature}")
    if not 0 <= top_k <= min(V, MAX_ENTRIES):
        raise ValueError(f"top_k must be in [0, min({MAX_ENTRIES}, V = {V})], got {top_k}")
    return (tokens if tokens.dim() == 1 else tokens.reshape(-1)).contiguous()


def _results(out, top_k: int) -> TokenLogprobs:
    return TokenLogprobs(out[0], out[1], *(out[2:] if top_k else (None, None)))


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, temperature: float = 1.0, top_k: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Log-probabilities of tokens [...] under logits [..., V] that exist (module docstring); differentiable in
    ``logits``."""
    _check_student(logits, "logits", "token_logprobs")
    ids = _check(logits, tokens, logits.shape[-1], temperature, top_k)
    return _results(_token_logprobs(logits, ids, temperature, top_k, ignore_index), top_k)


def linear_token_logprobs(hidden: torch.Tensor, weight: torch.Tensor, tokens: torch.Tensor,
                          bias: Optional[torch.Tensor] = None, chunk_size: int = 8192, temperature: float = 1.0,
                          top_k: int = 0, ignore_index: int = -100) -> TokenLogprobs:
    """Fused lm_head projection + log-probabilities of tokens (module docstring).

    hidden [..., d], weight [V, d], tokens [...], bias [V] or None; differentiable in
    hidden, weight and bias.  d is a multiple of 8.  ``chunk_size`` bounds the
    backward's vocabulary band, as in ``cut_cross_entropy``.
    """
    _check_student(hidden, "hidden", "linear_token_logprobs")
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
    ids = _check(hidden, tokens, weight.shape[0], temperature, top_k)
    return _results(_linear_token_logprobs(hidden, weight, bias, ids, chunk_size, temperature, top_k, ignore_index),
                    top_k)
