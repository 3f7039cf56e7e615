"""The gradients of several leaves are tensors of their own: what a caller does to one in place leaves the others as they
are.  On meta tensors; test_gpu_gradients_apart.py has the numbers."""
import pytest
import torch

import chronicals_amd.ops  # noqa: F401  (registers the operators)

ops = torch.ops.chronicals_hip


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


def leaf(*shape, dtype=torch.float32):
    return meta(*shape, dtype=dtype).requires_grad_(True)


def apart(leaves):
    """Each leaf has a gradient of its shape and type, in a storage that no other one uses."""
    for v in leaves:
        assert v.grad.shape == v.shape and v.grad.dtype == v.dtype
    return len({v.grad.untyped_storage()._cdata for v in leaves}) == len(leaves)


SHAPES = [(16,), (12, 16), (3, 4, 16), (2, 3, 2, 16), (0, 16), (2, 0, 16)]


@pytest.mark.parametrize("weight", [True, False])
@pytest.mark.parametrize("rdtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_rms_norm(shape, rdtype, weight):
    x, r = leaf(*shape, dtype=torch.bfloat16), leaf(*shape, dtype=rdtype)
    w = leaf(16) if weight else None
    for used in ((0, 1), (0,), (1,)):
        x.grad = r.grad = None
        out = ops.rms_norm(x, w, r, 1e-6)
        sum(out[i].float().sum() for i in used).backward()
        assert apart([x, r] + ([w] if weight else [])), used


def test_rms_norm_of_one_leaf_twice():
    for shape in SHAPES:
        x = leaf(*shape)
        y, s = ops.rms_norm(x, None, x, 1e-6)
        (y.sum() + s.sum()).backward()
        assert x.grad.shape == x.shape


@pytest.mark.parametrize("shape", [(16,), (12, 16), (3, 4, 16)])
def test_the_others(shape):
    n = torch.Size(shape[:-1]).numel()
    x, w, b = leaf(*shape), leaf(16), leaf(16)
    ops.layer_norm(x, w, b, 1e-5).sum().backward()
    assert apart([x, w, b])
    h, w, b, t = leaf(*shape), leaf(50, 16), leaf(50), meta(n, dtype=torch.int64)
    out = ops.linear_token_logprobs(h, w, b, t, 8192, 1.0, 0, -100)
    (out[0].sum() + out[1].sum()).backward()
    assert apart([h, w, b])
    h.grad = w.grad = b.grad = None
    ops.distill_linear(h, w, b, meta(n, 5), meta(n, 5, dtype=torch.int64), None, 8192, 1.0, 1.0, 0.0, -100, 1).backward()
    assert apart([h, w, b])


@pytest.mark.filterwarnings("ignore:Using backward")
@pytest.mark.parametrize("shape", SHAPES)
def test_rms_norm_of_one_type_as_an_addition(shape):
    """Asked for by torch.autograd.grad, the gradients of x and of a residual of its type are one tensor, as those of
    x + residual are: nothing that looks like two."""
    for twice in (False, True):
        x, r = leaf(*shape), leaf(*shape)
        y, s = ops.rms_norm(x, None, r, 1e-6)
        gx, gr = torch.autograd.grad(y.sum() + s.sum(), [x, r], create_graph=twice)
        assert gx is gr and gx.requires_grad == twice
        y, s = ops.rms_norm(x, None, r, 1e-6)
        (y.sum() + s.sum()).backward(create_graph=twice)
        assert apart([x, r])
        x.grad = r.grad = None
