"""Layer norm, the distillation losses and top_logits as operators: their schemas and fakes, compiled, with hooks on what
they save, and where function transforms are refused."""
import pytest
import torch
from torch.library import opcheck

from tests.distill_common import labels, teacher

pytestmark = pytest.mark.gpu

HOW = (2.0, 0.5, 0.5)
N, V, D, K = 40, 600, 64, 5


def tensors(gpu, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(60)
    t, index = teacher(g, N, V, K, 0.2)
    return dict(x=torch.randn(N, V, generator=g).to(dtype).to(gpu), h=torch.randn(N, D, generator=g).to(dtype).to(gpu),
                w=(torch.randn(V, D, generator=g) * 0.1).to(dtype).to(gpu), b=torch.randn(V, generator=g).to(gpu),
                p=torch.randn(D, generator=g).to(dtype).to(gpu), t=t.to(gpu), i=index.to(gpu), lab=labels(g, N, V).to(gpu))


@pytest.mark.parametrize("reduction", [0, 1, 2])
def test_opcheck(gpu, reduction):
    ops = torch.ops.chronicals_hip
    v = tensors(gpu)
    go = torch.ones(N if reduction == 0 else 1, device=gpu)
    args = (v["x"], v["t"], v["i"], v["lab"], *HOW, -100, reduction)
    opcheck(ops.distill_logits_fwd.default, args)
    _, stats, n = ops.distill_logits_fwd(*args)
    opcheck(ops.distill_logits_bwd.default, (go, *args[:4], stats, n, *HOW, -100, reduction))
    args = (v["h"], v["w"], v["b"], v["t"], v["i"], v["lab"], *HOW, -100, reduction)
    opcheck(ops.distill_fwd.default, args)
    _, stats, kept, rows, n = ops.distill_fwd(*args)
    for needs in ((True, True, True, False, False), (True, False, False, True, False), (False, True, False, False, True)):
        opcheck(ops.distill_bwd.default, (go, *args[:5], stats, kept, rows, n, *HOW, reduction, 8192, *needs))


def test_kept_logits_are_whole(gpu):
    """What the forward keeps holds 0 where a row has no entry or no label, or does not count, whatever was in the memory
    before."""
    v = tensors(gpu)
    for lab, ce in ((v["lab"], 0.5), (v["lab"], 0.0), (None, 0.0)):
        junk = torch.full((N * (K + 1),), float("nan"), device=gpu)  # freed: the output's block, most likely
        del junk
        _, _, kept, rows, _ = torch.ops.chronicals_hip.distill_fwd(v["h"], v["w"], v["b"], v["t"], v["i"], lab, 2.0, 0.5,
                                                                   ce, -100, 1)
        counts = rows >= 0
        usable = torch.cat([v["i"] >= 0, (counts if ce else torch.zeros_like(counts))[:, None]], 1) & counts[:, None]
        x = v["h"].double() @ v["w"].double().t() + v["b"].double()
        label = torch.zeros_like(rows).long() if lab is None else lab.clamp(min=0)
        at = torch.cat([v["i"].clamp(min=0), label[:, None]], 1)
        want = torch.where(usable, x.gather(1, at), 0.0)
        # D products of fp32 and the bias, each off by 2^-24 of the magnitudes
        mag = (v["h"].double().abs() @ v["w"].double().abs().t() + v["b"].double().abs()).gather(1, at)
        assert (~usable).any() and not kept[~usable].any()
        assert ((kept.double() - want).abs() <= (D + 2) * 2.0 ** -24 * mag).all()


def test_opcheck_top_and_norm(gpu):
    ops = torch.ops.chronicals_hip
    v = tensors(gpu)
    opcheck(ops.top_logits.default, (v["x"], 7))
    for p in (v["p"], None):
        opcheck(ops.layer_norm_fwd.default, (v["h"], p, p, 1e-5))
        _, mean, rstd = ops.layer_norm_fwd(v["h"], p, p, 1e-5)
        for needs in ((True, True, True), (True, False, False), (False, True, False)):
            opcheck(ops.layer_norm_bwd.default, (v["h"], v["h"], p, mean, rstd, False, *needs))


def test_opcheck_differentiable(gpu):
    """Those made of the others: what a trace with static and with symbolic sizes computes, gradients included."""
    ops = torch.ops.chronicals_hip
    v = tensors(gpu)
    utils = ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic")
    x, h, w, p = (v[k].clone().requires_grad_(True) for k in ("x", "h", "w", "p"))
    opcheck(ops.layer_norm.default, (h.detach().view(4, 10, D).requires_grad_(True), p, None, 1e-5), test_utils=utils)
    opcheck(ops.distill_logits.default, (x, v["t"], v["i"], v["lab"], *HOW, -100, 1), test_utils=utils)
    opcheck(ops.distill_linear.default, (h, w, v["b"], v["t"], v["i"], v["lab"], 8192, *HOW, -100, 0), test_utils=utils)


@pytest.mark.parametrize("dynamic", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_compiled_step(gpu, dtype, dynamic):
    """A whole step in one graph: the same bits as without."""
    from chronicals_amd.kernels.distillation import LinearDistillationLoss, distillation_loss, top_logits
    from chronicals_amd.kernels.layer_norm import LayerNorm
    v = tensors(gpu, dtype)
    norm = LayerNorm(D, device=gpu, dtype=dtype)
    head = LinearDistillationLoss(chunk_size=8192, temperature=2.0, distill_weight=0.5, ce_weight=0.5)

    def step(h, w, x, full, lab):
        values, indices = top_logits(full, K)
        loss = head(norm(h), w, values, indices, lab)
        loss += distillation_loss(x, values, indices, lab, temperature=2.0, distill_weight=0.5, ce_weight=0.5)
        return loss
    torch._dynamo.reset()
    compiled = torch.compile(step, fullgraph=True, dynamic=dynamic, backend="aot_eager")
    for rows in (N, N - 3):
        results = []
        for f in (step, compiled):
            h, w, x = (v[k][:rows if k != "w" else None].clone().requires_grad_(True) for k in ("h", "w", "x"))
            norm.zero_grad(set_to_none=True)
            loss = f(h.view(1, rows, D), w, x.view(1, rows, V), v["x"][:rows].view(1, rows, V), v["lab"][:rows].view(1, rows))
            loss.backward()
            results.append([loss.detach(), h.grad, w.grad, x.grad, norm.weight.grad, norm.bias.grad])
        assert all(torch.equal(a, b) for a, b in zip(*results))


def test_saved_tensors_pass_hooks(gpu):
    """Activations kept on the host, as torch.autograd.graph.save_on_cpu does, and checkpointed ones."""
    from chronicals_amd.kernels.distillation import distillation_loss, linear_distillation_loss
    from chronicals_amd.kernels.layer_norm import layer_norm
    from torch.utils.checkpoint import checkpoint
    v = tensors(gpu, torch.float32)
    x, h, w, p = (v[k].clone().requires_grad_(True) for k in ("x", "h", "w", "p"))

    def f(h, w, p, x):
        return (linear_distillation_loss(layer_norm(h, p), w, v["t"], v["i"], v["lab"], ce_weight=0.5) +
                distillation_loss(x, v["t"], v["i"], v["lab"], ce_weight=0.5))
    leaves = [h, w, p, x]
    want = torch.autograd.grad(f(*leaves), leaves)
    with torch.autograd.graph.save_on_cpu():
        loss = f(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(loss, leaves)))
    loss = checkpoint(f, *leaves, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(loss, leaves)))


def test_saved_operands_changed_in_place_raise(gpu):
    from chronicals_amd.kernels.distillation import distillation_loss
    from chronicals_amd.kernels.layer_norm import layer_norm
    v = tensors(gpu, torch.float32)
    for shape in ((N, V), (4, 10, V)):
        x = v["x"].clone().requires_grad_(True)
        y = x * 1.0
        z = layer_norm(y.view(shape))
        with torch.no_grad():
            y += 1.0
        with pytest.raises(RuntimeError, match="inplace"):
            z.sum().backward()
        y = x * 1.0
        lead = shape[:-1]
        loss = distillation_loss(y.view(shape), v["t"].view(*lead, K), v["i"].view(*lead, K), v["lab"].view(lead))
        with torch.no_grad():
            y += 1.0
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()


def test_function_transforms_are_refused(gpu):
    from chronicals_amd.kernels.distillation import distillation_loss
    from chronicals_amd.kernels.layer_norm import layer_norm
    v = tensors(gpu, torch.float32)
    loss = lambda x: distillation_loss(x, v["t"], v["i"], v["lab"])  # noqa: E731
    for f in (loss, lambda x: layer_norm(x).sum()):
        with pytest.raises(RuntimeError):
            torch.func.grad(f)(v["x"])
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (v["x"],), (v["x"],))
        with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError):
            f(torch.autograd.forward_ad.make_dual(v["x"], v["x"]))
