"""Autograd of the differentiable operators on meta tensors: what a caller may do with a result."""
import pytest
import torch

import chronicals_amd.ops  # noqa: F401  (registers the operators)

ops = torch.ops.chronicals_hip


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


def leaf(*shape, dtype=torch.float32):
    return meta(*shape, dtype=dtype).requires_grad_(True)


def teacher():
    return meta(12, 5), meta(12, 5, dtype=torch.int64)


def norm(x):
    return ops.layer_norm(x, leaf(x.shape[-1], dtype=x.dtype), None, 1e-5)


def from_logits(x, reduction=1):
    return ops.distill_logits(x, *teacher(), None, 1.0, 1.0, 0.0, -100, reduction)


def from_head(h, w, reduction=1):
    return ops.distill_linear(h, w, None, *teacher(), None, 8192, 1.0, 1.0, 0.0, -100, reduction)


RESULTS = [lambda: norm(leaf(12, 16)), lambda: norm(leaf(3, 4, 16)), lambda: norm(leaf(16))]
RESULTS += [lambda r=r: from_logits(leaf(12, 50), r) for r in range(3)]
RESULTS += [lambda r=r: from_head(leaf(12, 16), leaf(50, 16), r) for r in range(3)]


@pytest.mark.parametrize("make", RESULTS)
def test_results_may_be_changed_in_place(make):
    """loss /= steps, loss += another, h += residual, as torch's own operators allow."""
    y = make()
    assert y.requires_grad and not y._is_view()
    y /= 4
    y += 1
    y.sum().backward()
