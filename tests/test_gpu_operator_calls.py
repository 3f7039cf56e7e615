"""What callers do with the results of layer norm and of the distillation losses."""
import pytest
import torch

from tests.distill_common import labels, teacher

pytestmark = pytest.mark.gpu


def inputs(gpu, dtype=torch.float32, B=2, S=9, d=64, V=500, K=6):
    g = torch.Generator().manual_seed(50)
    t, index = teacher(g, B * S, V, K, 0.2)
    return dict(x=torch.randn(B, S, V, generator=g).to(dtype).to(gpu), h=torch.randn(B, S, d, generator=g).to(dtype).to(gpu),
                w=(torch.randn(V, d, generator=g) * 0.1).to(dtype).to(gpu), t=t.view(B, S, K).to(gpu),
                index=index.view(B, S, K).to(gpu), lab=labels(g, B * S, V).view(B, S).to(gpu))


HOW = dict(temperature=2.0, distill_weight=0.5, ce_weight=0.5)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_losses_changed_in_place(gpu, reduction, dtype):
    from chronicals_amd.kernels.distillation import distillation_loss, linear_distillation_loss
    v = inputs(gpu, dtype)
    a = {k: v[k].clone().requires_grad_(True) for k in ("x", "h", "w")}

    def losses():
        return (distillation_loss(a["x"], v["t"], v["index"], v["lab"], reduction=reduction, **HOW),
                linear_distillation_loss(a["h"], a["w"], v["t"], v["index"], v["lab"], reduction=reduction, **HOW))
    plain = losses()
    want = torch.autograd.grad([loss.sum() / 4 for loss in plain], list(a.values()))
    for loss, p in zip(changed := losses(), plain):
        loss /= 4
        loss += 1.0
        assert torch.equal(loss, p.detach() / 4 + 1.0)
    changed[0].sum().backward()
    changed[1].sum().backward()
    assert all(torch.equal(p.grad, q) for p, q in zip(a.values(), want))


@pytest.mark.parametrize("shape", [(18, 64), (2, 9, 64), (64,)])
def test_layer_norm_changed_in_place(gpu, shape):
    from chronicals_amd.kernels.layer_norm import LayerNorm
    g = torch.Generator().manual_seed(51)
    x, r = (torch.randn(shape, generator=g).to(gpu) for _ in range(2))
    norm = LayerNorm(64, device=gpu)
    leaves = [x.requires_grad_(True), norm.weight, norm.bias]
    plain = norm(x)
    want = torch.autograd.grad((torch.relu(plain + r) * r).sum(), leaves)
    y = norm(x)
    y += r
    y.relu_()
    assert torch.equal(y, torch.relu(plain + r)) and y.shape == shape
    (y * r).sum().backward()
    assert all(torch.equal(p.grad, q) for p, q in zip(leaves, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_gradients_are_not_differentiated_again(gpu, dtype):
    """Taken with create_graph they have the same bits, and a penalty on them raises, also where the operands that were
    saved are copies."""
    from chronicals_amd.kernels.distillation import distillation_loss, linear_distillation_loss
    from chronicals_amd.kernels.layer_norm import layer_norm
    v = inputs(gpu, dtype)
    h, w, x = (v[k].requires_grad_(True) for k in ("h", "w", "x"))
    wide = v["x"].detach().permute(2, 1, 0).contiguous().permute(2, 1, 0).requires_grad_(True)
    assert wide.stride(-1) != 1
    cases = [(lambda: linear_distillation_loss(h, w, v["t"], v["index"], v["lab"], **HOW), [h, w]),
             (lambda: distillation_loss(x, v["t"], v["index"], v["lab"], **HOW), [x]),
             (lambda: distillation_loss(wide, v["t"], v["index"], v["lab"], **HOW), [wide]),
             (lambda: layer_norm(wide).square().mean(), [wide])]
    for f, leaves in cases:
        plain = torch.autograd.grad(f(), leaves)
        loss = f()
        grads = torch.autograd.grad(loss, leaves, create_graph=True)
        for leaf, p, g in zip(leaves, plain, grads):
            assert g.requires_grad and not p.requires_grad and torch.equal(g, p) and g.stride() == p.stride()
            with pytest.raises(RuntimeError, match="differentiated again"):
                torch.autograd.grad(loss + g.float().square().sum(), leaf, retain_graph=True)
