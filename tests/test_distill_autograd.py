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


def strided(*shape):
    """A leaf whose transpose has rows that are not contiguous: the operators work on a copy."""
    return leaf(*reversed(shape)), lambda v: v.t()


TWICE = {
    "norm": lambda: (x := leaf(12, 16), norm(x)),
    "norm of a copy": lambda: ((p := strided(12, 16))[0], norm(p[1](p[0]))),
    "norm, the weight": lambda: (w := leaf(16), ops.layer_norm(meta(12, 16), w, None, 1e-5)),
    "logits": lambda: (x := leaf(12, 50), from_logits(x)),
    "logits of a copy": lambda: ((p := strided(12, 50))[0], from_logits(p[1](p[0]), 0)),
}
for _dt in (torch.bfloat16, torch.float16, torch.float32):
    TWICE[f"hidden, {_dt}"] = lambda dt=_dt: (h := leaf(12, 16, dtype=dt), from_head(h, meta(50, 16, dtype=dt)))
    TWICE[f"weight, {_dt}"] = lambda dt=_dt: (w := leaf(50, 16, dtype=dt), from_head(meta(12, 16, dtype=dt), w))


@pytest.mark.parametrize("name", list(TWICE))
def test_gradients_are_not_differentiated_again(name):
    """A gradient taken with create_graph leads back to the input and raises there, alone or within another loss: it is
    never taken for a constant."""
    x, y = TWICE[name]()
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    assert g.requires_grad and g.shape == x.shape and g.dtype == x.dtype
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(g.float().square().sum(), x, retain_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        (y.sum() + g.float().square().sum()).backward()


def test_gradients_depend_on_the_incoming_gradient():
    x, up = leaf(12, 16), leaf(12, 16)
    (g,) = torch.autograd.grad(norm(x), x, up, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(g.sum(), up)


def test_first_gradients_have_no_graph():
    x = leaf(12, 16)
    (g,) = torch.autograd.grad(norm(x).sum(), x)
    assert not g.requires_grad
    norm(x).sum().backward()
    assert not x.grad.requires_grad
