"""A backward pass captured into a HIP graph while another graph of the same leaves lives on the default stream: refused
by layer norm and the distillation losses too; with that graph gone, or made on the capturing stream, it works."""
import gc

import pytest
import torch

from tests.distill_common import labels, teacher

pytestmark = pytest.mark.gpu

N, V, D, K = 24, 500, 64, 5
KINDS = ["norm", "norm, frozen", "norm without a bias", "norm, vectors", "logits", "logits, rows", "head", "head, frozen",
         "head, rows"]


def case(gpu, kind):
    """(the leaves, the loss of them)"""
    from chronicals_amd.kernels.distillation import distillation_loss, linear_distillation_loss
    from chronicals_amd.kernels.layer_norm import layer_norm
    g = torch.Generator().manual_seed(70)
    x, h, w, b, p, q = (torch.randn(*s, generator=g).to(gpu).requires_grad_(True)
                        for s in ((N, V), (N, D), (V, D), (V,), (D,), (D,)))
    t, i = (v.to(gpu) for v in teacher(g, N, V, K, 0.2))
    lab = labels(g, N, V).to(gpu)
    up = torch.randn(N, generator=g).to(gpu)
    v3 = torch.randn(2, N, D, generator=g).to(gpu).requires_grad_(True)
    return {
        "norm": ([h, p, q], lambda: (layer_norm(h, p, q) * up[:, None]).sum()),
        "norm, frozen": ([h], lambda: (layer_norm(h, p.detach(), q.detach()) * up[:, None]).sum()),
        "norm without a bias": ([h, p], lambda: (layer_norm(h, p) * up[:, None]).sum()),
        "norm, vectors": ([v3, p], lambda: (layer_norm(v3, p) * up[:, None]).sum()),
        "logits": ([x], lambda: distillation_loss(x, t, i, lab, 2.0, 0.5, 0.5)),
        "logits, rows": ([x], lambda: (distillation_loss(x, t, i, reduction="none") * up).sum()),
        "head": ([h, w, b], lambda: linear_distillation_loss(h, w, t, i, lab, b, ce_weight=0.5)),
        "head, frozen": ([h], lambda: linear_distillation_loss(h, w.detach(), t, i)),
        "head, rows": ([h, w], lambda: (linear_distillation_loss(h, w, t, i, reduction="none") * up).sum()),
    }[kind]


def warm_up(f):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()


@pytest.mark.parametrize("kind", KINDS)
def test_an_eager_graph_alive(gpu, kind):
    leaves, loss = case(gpu, kind)
    want = torch.autograd.grad(loss(), leaves)
    warm_up(lambda: torch.autograd.grad(loss(), leaves))
    kept = loss()
    with pytest.raises(RuntimeError, match="another graph of the same leaves"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(loss(), leaves)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(kept, leaves), want))
    del kept
    gc.collect()  # and what the error's traceback held
    replayed(leaves, loss)


def replayed(leaves, loss):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.autograd.grad(loss(), leaves)
    first = [v.detach().clone() for v in leaves]
    for scale in (1.0, 0.5, 2.0, 1.0):
        with torch.no_grad():
            for v, f in zip(leaves, first):
                v.copy_(f * scale)
        graph.replay()
        got = [v.clone() for v in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(loss(), leaves))), scale


@pytest.mark.parametrize("kind", ["norm", "logits", "head"])
def test_a_graph_alive_on_the_capturing_stream(gpu, kind):
    leaves, loss = case(gpu, kind)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kept = loss()
        want = torch.autograd.grad(kept, leaves, retain_graph=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = torch.autograd.grad(loss(), leaves)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(kept, leaves), want))
