"""Token log-probabilities and RMS norm as operators: their schemas and fakes, compiled, with hooks on what they save, and
where function transforms are refused."""
import gc

import pytest
import torch
from torch.library import opcheck

from tests.logprobs_common import tokens

pytestmark = pytest.mark.gpu

N, V, D, K = 40, 600, 64, 5


def tensors(gpu, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(60)
    return dict(x=torch.randn(N, V, generator=g).to(dtype).to(gpu), h=torch.randn(N, D, generator=g).to(dtype).to(gpu),
                w=(torch.randn(V, D, generator=g) * 0.1).to(dtype).to(gpu), b=torch.randn(V, generator=g).to(gpu),
                p=torch.randn(D, generator=g).to(dtype).to(gpu), r=torch.randn(N, D, generator=g).to(gpu),
                t=tokens(g, N, V).to(gpu), g=torch.randn(N, generator=g).to(gpu))


def test_opcheck_logprobs(gpu):
    ops = torch.ops.chronicals_hip
    v = tensors(gpu)
    for k in (0, K):
        args = (v["x"], v["t"], 0.9, k, -100)
        opcheck(ops.token_logprobs_fwd.default, args)
        stats = ops.token_logprobs_fwd(*args)[2]
        lin = (v["h"], v["w"], v["b"], v["t"], 0.9, k, -100)
        opcheck(ops.linear_token_logprobs_fwd.default, lin)
        lstats = ops.linear_token_logprobs_fwd(*lin)[2]
    for g, h in ((v["g"], v["g"]), (v["g"], None), (None, v["g"])):
        opcheck(ops.token_logprobs_bwd.default, (g, h, v["x"], v["t"], stats, 0.9, -100))
        for needs in ((True, True, True, False, False), (True, False, False, True, False), (False, True, False, False, True)):
            opcheck(ops.linear_token_logprobs_bwd.default, (g, h, *lin[:4], lstats, 0.9, -100, 8192, *needs))


def test_opcheck_norm(gpu):
    ops = torch.ops.chronicals_hip
    v = tensors(gpu)
    for p in (v["p"], None):
        for r in (v["r"], v["h"], None):
            opcheck(ops.rms_norm_fwd.default, (v["h"], p, r, 1e-6))
            for int8, group in ((False, 0), (True, 0), (False, 32), (True, 128)):
                opcheck(ops.rms_norm_quantized.default, (v["h"], p, r, 1e-6, int8, group), test_utils=(
                    "test_schema", "test_faketensor"))
            _, s, rstd = ops.rms_norm_fwd(v["h"], p, r, 1e-6)
            s = v["h"] if r is None else s
            for needs in ((True, True, p is not None), (True, False, False), (False, True, False)):
                opcheck(ops.rms_norm_bwd.default, (v["h"], None if r is None else s, s, p, rstd, False, *needs))


def test_opcheck_differentiable(gpu):
    """Those made of the others: what a trace with static and with symbolic sizes computes, gradients included."""
    ops = torch.ops.chronicals_hip
    v = tensors(gpu)
    utils = ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic")
    x, h, w, p, r = (v[k].clone().requires_grad_(True) for k in ("x", "h", "w", "p", "r"))
    opcheck(ops.rms_norm.default, (h.detach().view(4, 10, D).requires_grad_(True), p, r.detach().view(4, 10, D), 1e-6),
            test_utils=utils)
    opcheck(ops.rms_norm.default, (h, p, r, 1e-6), test_utils=utils)
    opcheck(ops.token_logprobs.default, (x, v["t"], 0.9, K, -100), test_utils=utils)
    opcheck(ops.linear_token_logprobs.default, (h, w, v["b"], v["t"], 8192, 0.9, 0, -100), test_utils=utils)


@pytest.mark.parametrize("dynamic", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_compiled_step(gpu, dtype, dynamic):
    """A whole step in one graph: the same bits as without."""
    from chronicals_amd.kernels.rms_norm import RMSNorm
    from chronicals_amd.kernels.token_logprobs import linear_token_logprobs, token_logprobs
    v = tensors(gpu, dtype)
    norm = RMSNorm(D, device=gpu, dtype=dtype)

    def step(h, r, w, x, t, g):
        y, s = norm(h, r)
        a = linear_token_logprobs(y, w, t, temperature=0.9)
        b = token_logprobs(x, t, top_k=K)
        kept = b.top_logprobs.detach().sum() + b.top_indices.sum()
        return -(g * a.logprobs).sum() - 0.01 * a.entropy.sum() + (g * b.logprobs).sum() + s.square().mean(), kept
    torch._dynamo.reset()
    compiled = torch.compile(step, fullgraph=True, dynamic=dynamic, backend="aot_eager")
    for rows in (N, N - 3):
        results = []
        for f in (step, compiled):
            h, w, x = (v[k][:rows if k != "w" else None].clone().requires_grad_(True) for k in ("h", "w", "x"))
            r = v["r"][:rows].clone().requires_grad_(True)
            norm.zero_grad(set_to_none=True)
            loss, kept = f(h.view(1, rows, D), r.view(1, rows, D), w, x.view(1, rows, V), v["t"][:rows].view(1, rows),
                           v["g"][:rows].view(1, rows))
            loss.backward()
            results.append([loss.detach(), kept, h.grad, r.grad, w.grad, x.grad, norm.weight.grad])
        assert all(torch.equal(a, b) for a, b in zip(*results))


def test_saved_tensors_pass_hooks(gpu):
    """Activations kept on the host, as torch.autograd.graph.save_on_cpu does, and checkpointed ones."""
    from chronicals_amd.kernels.rms_norm import rms_norm
    from chronicals_amd.kernels.token_logprobs import linear_token_logprobs, token_logprobs
    from torch.utils.checkpoint import checkpoint
    v = tensors(gpu, torch.float32)
    leaves = [v[k].clone().requires_grad_(True) for k in ("x", "h", "w", "p", "r")]

    def f(x, h, w, p, r):
        y, s = rms_norm(h, p, r)
        a, b = linear_token_logprobs(y, w, v["t"]), token_logprobs(x, v["t"])
        return sum(o.logprobs.sum() + o.entropy.sum() for o in (a, b)) + s.sum()
    want = torch.autograd.grad(f(*leaves), leaves)
    with torch.autograd.graph.save_on_cpu():
        loss = f(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(loss, leaves)))
    loss = checkpoint(f, *leaves, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(loss, leaves)))


def test_saved_operands_changed_in_place_raise(gpu):
    from chronicals_amd.kernels.token_logprobs import token_logprobs
    v = tensors(gpu, torch.float32)
    for shape in ((N, V), (4, 10, V)):
        x = v["x"].clone().requires_grad_(True)
        y = x * 1.0
        out = token_logprobs(y.view(shape), v["t"].view(shape[:-1]))
        with torch.no_grad():
            y += 1.0
        with pytest.raises(RuntimeError, match="inplace"):
            out.logprobs.sum().backward()


def test_function_transforms_are_refused(gpu):
    from chronicals_amd.kernels.rms_norm import rms_norm
    from chronicals_amd.kernels.token_logprobs import token_logprobs
    v = tensors(gpu, torch.float32)
    for f in (lambda x: token_logprobs(x, v["t"]).logprobs.sum(), lambda x: rms_norm(x).sum()):
        with pytest.raises(RuntimeError):
            torch.func.grad(f)(v["x"])
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (v["x"],), (v["x"],))
        with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError):
            f(torch.autograd.forward_ad.make_dual(v["x"], v["x"]))


def test_results_changed_in_place(gpu):
    from chronicals_amd.kernels.token_logprobs import linear_token_logprobs, token_logprobs
    v = tensors(gpu, torch.float32)
    for lead in ((N,), (4, 10)):
        a = {k: v[k].clone().requires_grad_(True) for k in ("x", "h", "w")}

        def outs():
            return (token_logprobs(a["x"].view(*lead, V), v["t"].view(lead)),
                    linear_token_logprobs(a["h"].view(*lead, D), a["w"], v["t"].view(lead)))
        want = torch.autograd.grad([(o.logprobs / 4 + o.entropy).sum() for o in outs()], list(a.values()))
        changed = outs()
        for o in changed:
            lp = o.logprobs
            lp /= 4
            lp += o.entropy
            lp.sum().backward()
        assert all(torch.equal(p.grad, q) for p, q in zip(a.values(), want))


def test_an_eager_graph_alive_while_a_backward_is_captured(gpu):
    """A step is captured while another graph of the same leaves lives: refused, where the engine would tie the capture
    to the default stream.  With that graph gone the capture works."""
    from chronicals_amd.kernels.rms_norm import rms_norm
    from chronicals_amd.kernels.token_logprobs import linear_token_logprobs, token_logprobs
    v = tensors(gpu, torch.float32)
    x, h, p, w = (v[k].clone().requires_grad_(True) for k in ("x", "h", "p", "w"))
    cases = [([x], lambda: token_logprobs(x, v["t"]).logprobs.sum()), ([h, p], lambda: rms_norm(h, p).sum()),
             ([h, w], lambda: linear_token_logprobs(h, w, v["t"]).entropy.sum())]
    for leaves, loss in cases:
        want = torch.autograd.grad(loss(), leaves)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(loss(), leaves)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        kept = loss()
        with pytest.raises(RuntimeError, match="another graph of the same leaves"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                torch.autograd.grad(loss(), leaves)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(kept, leaves), want))
        del kept
        gc.collect()  # and what the error's traceback held
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = torch.autograd.grad(loss(), leaves)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
