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


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_head_rounds_its_operands_to_bf16(gpu, dtype):
    """fp16 and fp32 hidden states and weights take part as bf16 rounds them; gradients come back in their types, and
    fp32 ones are not rounded again."""
    from chronicals_amd.kernels.distillation import linear_distillation_loss
    g = torch.Generator().manual_seed(52)
    N, V, d, K = 300, 2000, 72, 8
    h, w, b = (v.to(dtype).to(gpu) for v in (torch.randn(N, d, generator=g), torch.randn(V, d, generator=g) * 0.1,
                                             torch.randn(V, generator=g)))
    t, index = (v.to(gpu) for v in teacher(g, N, V, K))
    lab = labels(g, N, V).to(gpu)

    def run(h, w, b):
        leaves = [v.clone().requires_grad_(True) for v in (h, w, b)]
        loss = linear_distillation_loss(leaves[0], leaves[1], t, index, lab, leaves[2], **HOW)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]
    h16, w16 = h.bfloat16(), w.bfloat16()
    assert not torch.equal(h16.to(dtype), h) and not torch.equal(w16.to(dtype), w)
    got = run(h, w, b)
    assert [v.dtype for v in got] == [torch.float32, dtype, dtype, dtype]
    # of the rounded values in the same types: the same bits
    same = run(h16.to(dtype), w16.to(dtype), b)
    assert all(torch.equal(p, q) for p, q in zip(got, same))
    # in bf16: the same products, rounded to bf16 at the end
    low = run(h16, w16, b)
    assert torch.equal(low[0], got[0]) and torch.equal(low[3], got[3])
    for p, q in zip(low[1:3], got[1:3]):
        if dtype == torch.float32:
            assert torch.equal(p, q.bfloat16())
        else:  # the fp32 result was rounded to fp16 on one side and to bf16 on the other
            tol = (2.0 ** -8 + 2.0 ** -11) * p.float().abs() + 2.0 ** -25
            assert ((p.float() - q.float()).abs() <= tol).all()
    # and against 64 bits of the operands as they were given: each logit is off by
    # 2^-8 of d products twice over, which moves a loss by as much at T and at 1
    hd, wd = h.double(), w.double()
    z = hd @ wd.t() + b.double()
    lp = torch.log_softmax(z / 2, 1).gather(1, index)
    lq = torch.log_softmax(t.double() / 2, 1)
    keep = lab != -100
    kd = 4 * (lq.exp() * (lq - lp)).sum(1)
    ce = torch.logsumexp(z, 1) - z.gather(1, lab.clamp(min=0)[:, None])[:, 0]
    want = ((0.5 * kd + 0.5 * ce) * keep).sum() / keep.sum()
    delta = ((2 * 2.0 ** -8 + 2.0 ** -16) * (hd.abs() @ wd.abs().t()).amax(1)) + 2.0 ** -20 * z.abs().amax(1)
    # d(0.5 T^2 KL) is 0.5 T (p - q) of total weight 2, and 0.5 (p - 1) likewise
    bound = ((0.5 * 2 * 2 + 0.5 * 2) * delta * keep).sum() / keep.sum() + 2.0 ** -13 * (1 + want)
    assert abs(got[0].double() - want) <= bound
