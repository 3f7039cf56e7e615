"""What the distillation, top-logits and layer-norm entry points refuse, and their schemas: without a GPU."""
import ctypes

import pytest
import torch

from chronicals_amd import _lib
from chronicals_amd.kernels import distillation as D
from chronicals_amd.kernels.layer_norm import LayerNorm, layer_norm

OPS = ("distill_logits_fwd", "distill_logits_bwd", "distill_fwd", "distill_bwd", "top_logits", "layer_norm_fwd",
       "layer_norm_bwd")


def meta(*shape, dtype=torch.float32):
    """A tensor that passes for a device tensor in the entry points' own checks."""
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.fixture
def on_device(monkeypatch):
    """Meta tensors count as device tensors: the checks behind the first one run, and the operators' fakes."""
    monkeypatch.setattr(D, "_check_student", _without_device(D._check_student))


def _without_device(check):
    class Seen:
        is_cuda = True

        def __init__(self, t):
            self.t = t

        def __getattr__(self, name):
            return getattr(self.t, name)
    return lambda x, name, what: check(Seen(x), name, what)


def test_host_tensors_are_refused():
    x, t, i = torch.zeros(2, 10), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="HIP devices"):
        D.distillation_loss(x, t, i)
    with pytest.raises(RuntimeError, match="HIP devices"):
        D.linear_distillation_loss(x, torch.zeros(5, 10), t, i)
    with pytest.raises(RuntimeError, match="HIP devices"):
        D.top_logits(x, 2)
    with pytest.raises(RuntimeError, match="HIP devices"):
        layer_norm(x)
    with pytest.raises(RuntimeError, match=r"\[\.\.\., 8\]"):
        LayerNorm(8)(x)


GOOD = dict(teacher_logits=(4, 3), teacher_indices=(4, 3))
BAD = [
    (dict(teacher_logits=meta(3, 3)), RuntimeError, "teacher_logits must be"),
    (dict(teacher_indices=meta(4, 2, dtype=torch.int64)), RuntimeError, "teacher_indices must have the shape"),
    (dict(teacher_indices=meta(4, 3)), RuntimeError, "int64 or int32"),
    (dict(teacher_logits=meta(4, 3, dtype=torch.float64)), RuntimeError, "not supported"),
    (dict(teacher_logits=meta(4, 257), teacher_indices=meta(4, 257, dtype=torch.int64)), RuntimeError, "1 to 256"),
    (dict(teacher_logits=meta(4, 0), teacher_indices=meta(4, 0, dtype=torch.int64)), RuntimeError, "1 to 256"),
    (dict(teacher_logits=torch.zeros(4, 3)), RuntimeError, "device"),
    (dict(labels=meta(5, dtype=torch.int64)), RuntimeError, "5 elements"),
    (dict(labels=meta(4)), RuntimeError, "labels must be int64"),
    (dict(labels=torch.zeros(4, dtype=torch.int64)), RuntimeError, "device"),
    (dict(ce_weight=0.5), ValueError, "needs labels"),
    (dict(temperature=0.0), ValueError, "temperature"),
    (dict(temperature=float("nan")), ValueError, "temperature"),
    (dict(temperature=1e4), ValueError, "temperature"),
    (dict(reduction="median"), ValueError, "reduction"),
]


@pytest.mark.parametrize("bad,error,text", BAD)
def test_refusals(on_device, bad, error, text):
    kw = dict(teacher_logits=meta(4, 3), teacher_indices=meta(4, 3, dtype=torch.int64))
    kw.update(bad)
    with pytest.raises(error, match=text):
        D.distillation_loss(meta(4, 100), **kw)
    with pytest.raises(error, match=text):
        D.linear_distillation_loss(meta(4, 64), meta(100, 64), **kw)


def test_refusals_of_the_head(on_device):
    t = dict(teacher_logits=meta(4, 3), teacher_indices=meta(4, 3, dtype=torch.int64))
    for h, w, b, text in ((meta(4, 64), meta(100, 32), None, "does not match"),
                          (meta(4, 64), meta(100), None, "must be \\[vocab_size, hidden_dim\\]"),
                          (meta(4, 64), meta(100, 64, dtype=torch.float64), None, "not supported"),
                          (meta(4, 64), meta(100, 64), meta(99), "bias must be"),
                          (meta(4, 64), torch.zeros(100, 64), None, "same device")):
        with pytest.raises(RuntimeError, match=text):
            D.linear_distillation_loss(h, w, bias=b, **t)
    for k in (0, 11, 257):
        with pytest.raises(ValueError, match="k must be in"):
            D.top_logits(meta(2, 10 if k < 257 else 1000), k)
    with pytest.raises(RuntimeError, match="not supported"):
        D.top_logits(meta(2, 10, dtype=torch.int32), 3)
    with pytest.raises(ValueError, match="reduction"):
        D.DistillationLoss(reduction="median")
    with pytest.raises(ValueError, match="reduction"):
        D.LinearDistillationLoss(reduction="median")


@pytest.mark.parametrize("name", OPS)
def test_operators_are_traceable(name):
    op = getattr(torch.ops.chronicals_hip, name).default
    assert torch.Tag.pt2_compliant_tag in op.tags
    assert " int " not in str(op._schema)


def test_fakes():
    ops = torch.ops.chronicals_hip
    x, t, i = meta(6, 50, dtype=torch.bfloat16), meta(6, 4), meta(6, 4, dtype=torch.int64)
    loss, stats, n = ops.distill_logits_fwd(x, t, i, None, 1.0, 1.0, 0.0, -100, 1)
    assert loss.shape == (1,) and stats.shape == (6, 4) and n.dtype == torch.int32
    dx = ops.distill_logits_bwd(loss, x, t, i, None, stats, n, 1.0, 1.0, 0.0, -100, 1)
    assert dx.shape == x.shape and dx.dtype == x.dtype
    h, w = meta(6, 16, dtype=torch.bfloat16), meta(50, 16, dtype=torch.bfloat16)
    loss, stats, kept, rows, n = ops.distill_fwd(h, w, None, t, i, None, 1.0, 1.0, 0.0, -100, 0)
    assert loss.shape == (6,) and stats.shape == (6, 2) and kept.shape == (6, 5) and rows.dtype == torch.int32
    dh, dw, db = ops.distill_bwd(loss, h, w, None, t, i, stats, kept, rows, n, 1.0, 1.0, 0.0, 0, 8192, True, True, False,
                                 False, True)
    assert dh.shape == h.shape and dw.dtype == torch.float32 and db.shape == (0,)
    v, at = ops.top_logits(x, 3)
    assert v.shape == at.shape == (6, 3) and v.dtype == x.dtype and at.dtype == torch.int64
    y, mean, rstd = ops.layer_norm_fwd(x, None, None, 1e-5)
    assert y.shape == x.shape and mean.shape == rstd.shape == (6,)
    dx, dw, db = ops.layer_norm_bwd(y, x, None, mean, rstd, True, True, True, False)
    assert dx.dtype == torch.bfloat16 and dw.shape == (50,) and dw.dtype == torch.float32 and db.shape == (0,)


def test_differentiable_operators_trace():
    """A trace of forward and backward holds the operators underneath, with sizes that stay symbolic."""
    from torch.fx.experimental.proxy_tensor import make_fx
    ops = torch.ops.chronicals_hip

    def f(x, h, w, b, t, i, lab):
        n = ops.layer_norm(h, w[0], None, 1e-5)
        loss = ops.distill_linear(n, w, b, t, i, lab, 8192, 2.0, 0.5, 0.5, -100, 1)
        loss = loss + ops.distill_logits(x, t, i, None, 1.0, 1.0, 0.0, -100, 1)
        return torch.autograd.grad(loss, [x, h, w, b])

    def leaf(*shape):
        return meta(*shape).requires_grad_(True)
    args = (leaf(3, 4, 50), leaf(3, 4, 16), leaf(50, 16), leaf(50), meta(12, 5), meta(12, 5, dtype=torch.int64),
            meta(12, dtype=torch.int64))
    for mode in ("fake", "symbolic"):
        graph = make_fx(f, tracing_mode=mode)(*args).graph
        called = [str(n.target) for n in graph.nodes if "chronicals_hip" in str(n.target)]
        assert sorted(c.split(".")[1] for c in called) == ["distill_bwd", "distill_fwd", "distill_logits_bwd",
                                                           "distill_logits_fwd", "layer_norm_bwd", "layer_norm_fwd"]


# ---------------------------------------------------------------------------
# the C entry points: refusals come before any call to the device
# ---------------------------------------------------------------------------

P = ctypes.c_void_p(4096)  # an aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def a_teacher(**kw):
    f = dict(logits=4096, indices=4096, entries=4, logits_dtype=1, indices_int64=1, temperature=1.0, distill_weight=1.0,
             ce_weight=0.0)
    f.update(kw)
    return ctypes.byref(_lib.Teacher(**f))


TEACHERS = [(dict(entries=0), b"entries"), (dict(entries=257), b"entries"), (dict(logits_dtype=7), b"teacher's logits"),
            (dict(temperature=0.0), b"temperature"), (dict(temperature=float("nan")), b"temperature"),
            (dict(temperature=float("inf")), b"temperature"), (dict(distill_weight=float("inf")), b"finite"),
            (dict(ce_weight=1.0), b"needs labels"), (dict(logits=None), b"null"), (dict(indices=None), b"null")]


@pytest.mark.parametrize("kw,text", TEACHERS)
def test_c_teachers(lib, kw, text):
    t = a_teacher(**kw)
    rcs = [lib.cce_distill_logits_forward(P, 1, 100, t, None, 0, 4, 100, -100, 1, P, P, P, P, 1 << 30, None)]
    assert text in lib.cce_last_error()
    rcs.append(lib.cce_distill_logits_backward(P, P, 1, 100, t, None, 0, P, P, 4, 100, -100, 1, P, 100, None))
    assert text in lib.cce_last_error()
    rcs.append(lib.cce_distill_forward(P, P, None, t, None, 0, 4, 64, 100, -100, 1, P, P, P, P, P, P, 1 << 30, None))
    assert text in lib.cce_last_error()
    assert rcs == [_lib.CCE_ERR_INVALID_ARG] * 3


def test_c_operands(lib):
    bad, small = _lib.CCE_ERR_INVALID_ARG, _lib.CCE_ERR_WORKSPACE
    t = a_teacher()
    odd = ctypes.c_void_p(4100)
    fwd, bwd = lib.cce_distill_logits_forward, lib.cce_distill_logits_backward
    assert fwd(P, 1, 100, None, None, 0, 4, 100, -100, 1, P, P, P, P, 1 << 30, None) == bad
    assert fwd(P, 1, 99, t, None, 0, 4, 100, -100, 1, P, P, P, P, 1 << 30, None) == bad
    assert fwd(P, 5, 100, t, None, 0, 4, 100, -100, 1, P, P, P, P, 1 << 30, None) == bad
    assert fwd(P, 1, 100, t, None, 0, 4, 100, -100, 3, P, P, P, P, 1 << 30, None) == bad
    assert fwd(None, 1, 100, t, None, 0, 4, 100, -100, 1, P, P, P, P, 1 << 30, None) == bad
    assert fwd(P, 1, 100, t, None, 0, 4, 100, -100, 1, P, odd, P, P, 1 << 30, None) == bad
    assert fwd(P, 1, 100, t, None, 0, 4, 100, -100, 1, P, P, P, P, 8, None) == small
    assert bwd(P, P, 1, 100, t, None, 0, P, P, 4, 100, -100, 1, P, 99, None) == bad   # P twice: in place
    assert bwd(P, P, 1, 100, t, None, 0, P, P, 4, 100, -100, 1, P, 100, None) == bad
    lin = lib.cce_distill_forward
    assert lin(P, P, None, t, None, 0, 4, 60, 100, -100, 1, P, P, P, P, P, P, 1 << 30, None) == bad
    assert lin(odd, P, None, t, None, 0, 4, 64, 100, -100, 1, P, P, P, P, P, P, 1 << 30, None) == bad
    assert lin(P, P, None, t, None, 0, 4, 64, 100, -100, 1, P, P, P, P, P, P, 8, None) == small
    back = lib.cce_distill_backward
    assert back(P, P, P, None, t, P, P, None, P, 4, 64, 100, 1, 0, P, 0, P, 0, None, P, 1 << 30, None) == bad
    assert back(P, P, P, None, t, P, P, P, P, 4, 64, 100, 1, 0, P, 0, P, 0, P, P, 1 << 30, None) == bad  # no bias
    assert back(P, P, P, None, t, P, P, P, P, 4, 64, 100, 1, 0, P, 0, P, 0, None, P, 8, None) == small
    assert back(P, P, P, None, t, P, P, P, P, 4, 64, 1 << 33, 1, 0, P, 0, P, 0, None, P, 1 << 30, None) == bad
    top = lib.cce_top_logits
    for V, k in ((100, 0), (100, 101), (1000, 257), (0, 1)):
        assert top(P, 1, V, 4, V, k, P, P, P, 1 << 30, None) == bad
    assert top(P, 1, 99, 4, 100, 3, P, P, P, 1 << 30, None) == bad
    assert top(None, 1, 100, 4, 100, 3, P, P, P, 1 << 30, None) == bad
    assert top(P, 1, 1 << 17, 4, 1 << 17, 3, P, P, P, 8, None) == small
    norm, back = lib.cce_layer_norm_forward, lib.cce_layer_norm_backward
    assert norm(P, 0, 63, P, P, 0, 4, 64, 1e-5, P, P, P, None) == bad
    assert norm(P, 0, 64, P, P, 2, 4, 64, 1e-5, P, P, P, None) == bad
    assert norm(P, 0, 64, P, P, 0, 4, 0, 1e-5, P, P, P, None) == bad
    assert norm(P, 0, 64, P, P, 0, 4, 64, -1.0, P, P, P, None) == bad
    assert norm(P, 0, 64, P, P, 0, 4, 64, float("nan"), P, P, P, None) == bad
    assert norm(P, 0, 64, P, P, 0, 4, 64, 1e-5, None, P, P, None) == bad
    assert back(P, P, 0, 64, P, 0, P, P, 4, 64, P, P, P, P, 8, None) == small
    assert back(None, P, 0, 64, P, 0, P, P, 4, 64, P, P, P, P, 1 << 30, None) == bad


def test_source_hash_follows_the_parts(tmp_path, monkeypatch):
    from chronicals_amd import build
    text = open(build.SRC).read()
    for part in build.PARTS:
        assert f'#include "{part.rsplit("/", 1)[1]}"' in text
    base, torch_base = build.source_hash(), build.source_hash((build.TORCH_SRC, build.HEADER))
    edited = tmp_path / "distill.h"
    edited.write_text(open(build.PARTS[0]).read() + "// edit\n")
    monkeypatch.setattr(build, "PARTS", (str(edited), *build.PARTS[1:]))
    assert build.source_hash() != base
    assert build.source_hash((build.TORCH_SRC, build.HEADER)) == torch_base


def test_c_workspaces(lib):
    def size(fn, *args):
        out = ctypes.c_size_t(0)
        assert fn(*args, ctypes.byref(out)) == 0, lib.cce_last_error()
        return out.value
    # a few floats per row and split, never the logits
    assert 0 < size(lib.cce_distill_logits_workspace_bytes, 4096, 151936, 1) < 4096 * 64
    assert size(lib.cce_distill_logits_workspace_bytes, 0, 100, 0) > 0
    # beside the cross-entropy's forward: a third sum per split and two numbers per row
    ce = _lib.forward_workspace_bytes(4096, 896, 151936, 1, 1)
    assert ce < size(lib.cce_distill_forward_workspace_bytes, 4096, 896, 151936, 1) <= 2 * ce + 4096 * 16
    # beside its backward: a column and a value per entry
    ce = _lib.backward_workspace_bytes(4096, 896, 151936, 8192, True, True)
    kd = size(lib.cce_distill_backward_workspace_bytes, 4096, 896, 151936, 64, 8192, 1, 0, 1, 0)
    assert 4096 * 65 * 8 <= kd - ce <= 4096 * 65 * 8 + 1024
    assert size(lib.cce_layer_norm_backward_workspace_bytes, 0, 64) > 0
    # parts of the parameters' gradients: little next to long rows, bounded for the longest
    assert size(lib.cce_layer_norm_backward_workspace_bytes, 1 << 20, 1 << 20) <= (128 << 20) + 1024
    assert size(lib.cce_layer_norm_backward_workspace_bytes, 1 << 20, 4096) == 768 * 4096 * 8
    # the splits' candidates where there are few rows, nothing else
    assert size(lib.cce_top_logits_workspace_bytes, 4096, 151936, 64) == 0
    assert 0 < size(lib.cce_top_logits_workspace_bytes, 3, 151936, 64) <= 3 * 2048 * 8
    out = ctypes.c_size_t(0)
    assert lib.cce_distill_backward_workspace_bytes(8, 64, 100, 257, 0, 1, 0, 1, 0, ctypes.byref(out)) != 0
    assert lib.cce_distill_forward_workspace_bytes(8, 60, 100, 1, ctypes.byref(out)) != 0
