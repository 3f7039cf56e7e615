"""RMS norm's gradients of x and of a residual of its type, as leaves: accumulated, changed in place, in a checkpoint.

Every expected number is the gradient that one call of torch.autograd.grad over 2-D rows gives, whose values
test_gpu_rms_norm.py checks against 64 bits; sums of two equal fp32 or bf16 numbers are exact."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu

SHAPES = [(40,), (6, 40), (2, 3, 40), (3, 1, 2, 40)]
TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)]


def rms_norm(*args):
    from chronicals_amd.kernels.rms_norm import rms_norm as f
    return f(*args)


def operands(gpu, shape, dtype, rdtype=None):
    g = torch.Generator().manual_seed(len(shape))
    x, r, w = (torch.randn(*s, generator=g) for s in (shape, shape, shape[-1:]))
    ups = [torch.randn(*shape, generator=g) for _ in range(2)]
    return ([v.to(t).to(gpu).requires_grad_(True) for v, t in zip((x, w, r), (dtype, dtype, rdtype or dtype))],
            [v.to(t).to(gpu) for v, t in zip(ups, (dtype, rdtype or dtype))])


def expected(leaves, ups):
    x, w, r = (v.detach().view(-1, v.shape[-1]).requires_grad_(True) if i != 1 else v for i, v in enumerate(leaves))
    outs = rms_norm(x, w, r)
    grads = torch.autograd.grad(outs, [x, w, r], [u.view(x.shape) for u in ups])
    return [g.view(v.shape).clone() for g, v in zip(grads, leaves)]


def equal(leaves, want, times):
    return [torch.equal(v.grad, w * t) for v, w, t in zip(leaves, want, times)] == [True] * len(leaves)


@pytest.mark.parametrize("dtype,rdtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_accumulated(gpu, shape, dtype, rdtype):
    leaves, ups = operands(gpu, shape, dtype, rdtype)
    want = expected(leaves, ups)
    for times in (1, 2):
        torch.autograd.backward(rms_norm(*leaves), ups)
        assert equal(leaves, want, [times] * 3), times


def doubled(v):
    v.grad.mul_(2)


@pytest.mark.parametrize("shape", SHAPES)
def test_one_changed_in_place(gpu, shape):
    """As clipping, unscaling or a hook that runs after the accumulation does."""
    for changed in (0, 2):
        leaves, ups = operands(gpu, shape, torch.float32)
        want = expected(leaves, ups)
        torch.autograd.backward(rms_norm(*leaves), ups)
        leaves[changed].grad.mul_(4)
        assert equal(leaves, want, [4 if i == changed else 1 for i in range(3)])
        leaves, ups = operands(gpu, shape, torch.float32)
        leaves[changed].register_post_accumulate_grad_hook(doubled)
        torch.autograd.backward(rms_norm(*leaves), ups)
        assert equal(leaves, want, [2 if i == changed else 1 for i in range(3)])


@pytest.mark.parametrize("reentrant", [True, False])
@pytest.mark.parametrize("shape", SHAPES)
def test_checkpoint(gpu, shape, reentrant):
    leaves, ups = operands(gpu, shape, torch.float32)
    want = expected(leaves, ups)
    for times in (1, 2):
        torch.autograd.backward(checkpoint(rms_norm, *leaves, use_reentrant=reentrant), ups)
        assert equal(leaves, want, [times] * 3), times


@pytest.mark.parametrize("shape", SHAPES)
def test_what_comes_before(gpu, shape):
    """x and the residual of one leaf, or made of leaves by operators that hand their gradient on as it is."""
    leaves, ups = operands(gpu, shape, torch.float32)
    want = expected(leaves, ups)
    x, w, r = leaves
    a = torch.zeros_like(x).requires_grad_(True)
    for times in (1, 2):
        torch.autograd.backward(rms_norm(x + a, w, r + a), ups)
        assert equal(leaves, want, [times] * 3), times
        assert torch.equal(a.grad, want[0] * 2 * times)
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    y, s = rms_norm(x, w, x)
    (gx,) = torch.autograd.grad((y, s), x, ups, retain_graph=True)
    for times in (1, 2):
        torch.autograd.backward((y, s), ups, retain_graph=True)
        assert torch.equal(x.grad, gx * times)
    two = x.detach().requires_grad_(True), x.detach().requires_grad_(True)
    torch.autograd.backward(rms_norm(two[0], w, two[1]), ups)
    assert torch.equal(two[0].grad + two[1].grad, gx)
