"""What the token log-probabilities and the RMS norm refuse, their schemas, fakes and autograd: without a GPU."""
import ctypes

import pytest
import torch

from chronicals_amd import _lib
from chronicals_amd.kernels import rms_norm as R
from chronicals_amd.kernels import token_logprobs as L

ops = torch.ops.chronicals_hip
OPS = ("token_logprobs_fwd", "token_logprobs_bwd", "linear_token_logprobs_fwd", "linear_token_logprobs_bwd",
       "rms_norm_fwd", "rms_norm_quantized", "rms_norm_bwd")
I64 = torch.int64


def meta(*shape, dtype=torch.float32):
    """A tensor that passes for a device tensor in the entry points' own checks."""
    return torch.empty(shape, dtype=dtype, device="meta")


def leaf(*shape, dtype=torch.float32):
    return meta(*shape, dtype=dtype).requires_grad_(True)


class Seen:
    """A meta tensor that says it is on a device."""
    is_cuda = True

    def __init__(self, t):
        self.t = t

    def __getattr__(self, name):
        return getattr(self.t, name)


@pytest.fixture
def on_device(monkeypatch):
    """Meta tensors count as device tensors: the checks behind the first one run, and the operators' fakes."""
    student, norm = L._check_student, R._check
    monkeypatch.setattr(L, "_check_student", lambda x, name, what: student(Seen(x), name, what))
    monkeypatch.setattr(R, "_check", lambda x, *args: norm(Seen(x), *args))


def test_host_tensors_are_refused():
    x, t = torch.zeros(2, 16), torch.zeros(2, dtype=I64)
    for f in (lambda: L.token_logprobs(x, t), lambda: L.linear_token_logprobs(x, torch.zeros(5, 16), t),
              lambda: R.rms_norm(x), lambda: R.rms_norm_quantized(x)):
        with pytest.raises(RuntimeError, match="HIP devices"):
            f()
    with pytest.raises(RuntimeError, match=r"\[\.\.\., 8\]"):
        R.RMSNorm(8)(x)


@pytest.mark.parametrize("kw,error,text", [
    (dict(tokens=meta(5, dtype=I64)), RuntimeError, "tokens must be"),
    (dict(tokens=meta(4, 1, dtype=I64)), RuntimeError, "tokens must be"),
    (dict(tokens=meta(4)), RuntimeError, "int64 or int32"),
    (dict(tokens=torch.zeros(4, dtype=I64)), RuntimeError, "device"),
    (dict(temperature=0.0), ValueError, "temperature"),
    (dict(temperature=float("nan")), ValueError, "temperature"),
    (dict(temperature=1e4), ValueError, "temperature"),
    (dict(top_k=-1), ValueError, "top_k"),
    (dict(top_k=101), ValueError, "top_k"),
])
def test_refusals(on_device, kw, error, text):
    kw = {"tokens": meta(4, dtype=I64), **kw}
    with pytest.raises(error, match=text):
        L.token_logprobs(meta(4, 100), **kw)
    with pytest.raises(error, match=text):
        L.linear_token_logprobs(meta(4, 64), meta(100, 64), **kw)


def test_refusals_of_operands(on_device):
    t = meta(4, dtype=I64)
    with pytest.raises(ValueError, match="top_k"):
        L.token_logprobs(meta(4, 1000), t, top_k=257)
    with pytest.raises(RuntimeError, match="not supported"):
        L.token_logprobs(meta(4, 100, dtype=torch.float64), t)
    for h, w, b, text in ((meta(4, 64), meta(100, 32), None, "does not match"),
                          (meta(4, 64), meta(100), None, "must be \\[vocab_size, hidden_dim\\]"),
                          (meta(4, 64), meta(100, 64, dtype=torch.float64), None, "not supported"),
                          (meta(4, 64), meta(100, 64), meta(99), "bias must be"),
                          (meta(4, 64), meta(100, 64), torch.zeros(100), "same device"),
                          (meta(4, 64), torch.zeros(100, 64), None, "same device")):
        with pytest.raises(RuntimeError, match=text):
            L.linear_token_logprobs(h, w, t, b)


@pytest.mark.parametrize("kw,error,text", [
    (dict(x=meta(4, 16, dtype=torch.float64)), RuntimeError, "not supported"),
    (dict(x=meta(4, 0)), RuntimeError, "D >= 1"),
    (dict(eps=-1.0), ValueError, "eps"),
    (dict(eps=float("inf")), ValueError, "eps"),
    (dict(weight=meta(15)), RuntimeError, "weight must be"),
    (dict(weight=torch.zeros(16)), RuntimeError, "same device"),
    (dict(weight=meta(16, dtype=torch.float16)), RuntimeError, "weight must have"),
    (dict(residual=meta(4, 15)), RuntimeError, "x's shape"),
    (dict(residual=meta(16)), RuntimeError, "x's shape"),
    (dict(residual=torch.zeros(4, 16)), RuntimeError, "same device"),
    (dict(residual=meta(4, 16, dtype=torch.float16)), RuntimeError, "residual must have"),
])
def test_refusals_of_the_norm(on_device, kw, error, text):
    kw = {"x": meta(4, 16, dtype=torch.bfloat16), **kw}
    for f in (R.rms_norm, R.rms_norm_quantized):
        with pytest.raises(error, match=text):
            f(**kw)


def test_refusals_of_the_quantized_norm(on_device):
    x = meta(4, 16)
    with pytest.raises(ValueError, match="dtype must be"):
        R.rms_norm_quantized(x, dtype=torch.uint8)
    for group in (0, 16, 96, 512):
        with pytest.raises(ValueError, match="group_size"):
            R.rms_norm_quantized(x, group_size=group)


@pytest.mark.parametrize("name", OPS)
def test_operators_are_traceable(name):
    op = getattr(ops, name).default
    assert torch.Tag.pt2_compliant_tag in op.tags
    assert " int " not in str(op._schema)


def test_fakes():
    x, t = meta(6, 50, dtype=torch.bfloat16), meta(6, dtype=I64)
    h, w = meta(6, 16, dtype=torch.bfloat16), meta(50, 16, dtype=torch.bfloat16)
    for k in (0, 3):
        for out in (ops.token_logprobs_fwd(x, t, 1.0, k, -100), ops.linear_token_logprobs_fwd(h, w, None, t, 1.0, k, -100)):
            assert [tuple(v.shape) for v in out] == [(6,), (6,), (6, 4), (6, k), (6, k)]
            assert out[4].dtype == I64 and all(v.dtype == torch.float32 for v in out[:4])
    lp, H, stats = out[:3]
    dx = ops.token_logprobs_bwd(lp, None, x, t, stats, 1.0, -100)
    assert dx.shape == x.shape and dx.dtype == x.dtype
    dh, dw, db = ops.linear_token_logprobs_bwd(lp, H, h, w, None, t, stats, 1.0, -100, 8192, True, True, False, False, True)
    assert dh.shape == h.shape and dh.dtype == h.dtype and dw.dtype == torch.float32 and db.shape == (0,)
    y, s, rstd = ops.rms_norm_fwd(x, None, None, 1e-6)
    assert y.shape == x.shape and s.shape == (0,) and rstd.shape == (6,)
    y, s, rstd = ops.rms_norm_fwd(x, None, meta(6, 50), 1e-6)
    assert s.dtype == torch.float32 and s.shape == x.shape
    dx, dr, dw = ops.rms_norm_bwd(y, None, s, meta(50), rstd, True, True, True, True)
    assert dx.dtype == torch.bfloat16 and dr.dtype == dw.dtype == torch.float32 and dw.shape == (50,)
    q, scales, s = ops.rms_norm_quantized(x, None, x, 1e-6, False, 32)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scales.shape == (6, 2) and s.dtype == x.dtype
    q, scales, s = ops.rms_norm_quantized(x, None, None, 1e-6, True, 0)
    assert q.dtype == torch.int8 and scales.shape == (6,)


def test_shapes_of_results(on_device):
    out = L.token_logprobs(meta(2, 3, 50), meta(2, 3, dtype=I64), top_k=4)
    assert out.logprobs.shape == out.entropy.shape == (2, 3) and out.top_logprobs.shape == out.top_indices.shape == (2, 3, 4)
    out = L.linear_token_logprobs(meta(16), meta(50, 16), meta(dtype=I64))
    assert out.logprobs.shape == () and out.top_logprobs is None and out.top_indices is None
    y, s = R.rms_norm(meta(2, 3, 16), None, meta(2, 3, 16))
    assert y.shape == s.shape == (2, 3, 16)
    q, scales, s = R.rms_norm_quantized(meta(2, 3, 100), None, meta(2, 3, 100), group_size=32)
    assert q.shape == s.shape == (2, 3, 100) and scales.shape == (2, 3, 4)
    q, scales = R.rms_norm_quantized(meta(100))
    assert scales.shape == ()


def test_differentiable_operators_trace():
    """A trace of forward and backward holds the operators underneath, with sizes that stay symbolic."""
    from torch.fx.experimental.proxy_tensor import make_fx

    def f(x, h, w, b, r, t):
        n, s = ops.rms_norm(h, w[0], r, 1e-6)
        out = ops.linear_token_logprobs(n, w, b, t, 8192, 0.9, 0, -100)
        loss = out[0].sum() - out[1].sum() + s.sum() + ops.token_logprobs(x, t, 1.0, 2, -100)[0].sum()
        return torch.autograd.grad(loss, [x, h, w, b, r])

    args = (leaf(3, 4, 50), leaf(3, 4, 16), leaf(50, 16), leaf(50), leaf(3, 4, 16), meta(12, dtype=I64))
    for mode in ("fake", "symbolic"):
        graph = make_fx(f, tracing_mode=mode)(*args).graph
        called = [str(n.target) for n in graph.nodes if "chronicals_hip" in str(n.target)]
        assert sorted(c.split(".")[1] for c in called) == sorted(
            ["token_logprobs_fwd", "token_logprobs_bwd", "linear_token_logprobs_fwd", "linear_token_logprobs_bwd",
             "rms_norm_fwd", "rms_norm_bwd"])


RESULTS = [lambda i=i, s=s: ops.token_logprobs(leaf(*s, 50), meta(12, dtype=I64), 1.0, 2, -100)[i]
           for i in (0, 1) for s in ((12,), (3, 4))]
RESULTS += [lambda i=i, s=s: ops.linear_token_logprobs(leaf(*s, 16), leaf(50, 16), None, meta(12, dtype=I64), 8192, 1.0, 0,
                                                       -100)[i] for i in (0, 1) for s in ((12,), (3, 4))]
RESULTS += [lambda s=s: ops.rms_norm(leaf(*s, 16), leaf(16), None, 1e-6)[0] for s in ((12,), (3, 4), ())]
RESULTS += [lambda: ops.rms_norm(leaf(12, 16), leaf(16), leaf(12, 16), 1e-6)[0]]


@pytest.mark.parametrize("make", RESULTS)
def test_results_may_be_changed_in_place(make):
    y = make()
    assert y.requires_grad and not y._is_view()
    y /= 4
    y += 1
    y.sum().backward()


def test_gradients_are_not_differentiated_again():
    x, h, w, r, up = leaf(12, 50), leaf(12, 16), leaf(50, 16), leaf(12, 16), leaf(12)
    t = meta(12, dtype=I64)
    a, b = ops.token_logprobs(x, t, 1.0, 0, -100), ops.linear_token_logprobs(h, w, None, t, 8192, 1.0, 0, -100)
    y, s = ops.rms_norm(h, None, r, 1e-6)
    for out, leaves in ((a[0], [x]), (a[1], [x]), (b[0], [h, w]), (b[1], [h, w]), (y, [h, r]), (s, [h, r])):
        for v in leaves:
            (g,) = torch.autograd.grad(out.sum(), v, create_graph=True)
            assert g.requires_grad and g.shape == v.shape and g.dtype == v.dtype
            with pytest.raises(RuntimeError, match="differentiated again"):
                torch.autograd.grad(g.sum(), v, retain_graph=True)
    (g,) = torch.autograd.grad(a[1], x, up, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(g.sum(), up)


# ---------------------------------------------------------------------------
# the C entry points: refusals come before any call to the device
# ---------------------------------------------------------------------------

P = ctypes.c_void_p(4096)  # an aligned address that nothing reads
ODD = ctypes.c_void_p(4100)
BAD, SMALL, BIG = _lib.CCE_ERR_INVALID_ARG, _lib.CCE_ERR_WORKSPACE, 1 << 40


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_c_token_logprobs(lib):
    def fwd(logits=P, dtype=1, ld=100, tokens=P, N=4, V=100, T=1.0, k=0, lp=P, h=P, stats=P, tl=P, ti=P, ws=P, n=BIG):
        return lib.cce_token_logprobs_forward(logits, dtype, ld, tokens, 1, N, V, -100, T, k, lp, h, stats, tl, ti, ws, n,
                                              None)
    for kw in (dict(logits=None), dict(dtype=3), dict(ld=99), dict(tokens=None), dict(N=-1), dict(V=0), dict(T=0.0),
               dict(T=float("nan")), dict(T=float("inf")), dict(k=-1), dict(k=101), dict(V=1000, ld=1000, k=257),
               dict(lp=None), dict(h=None), dict(stats=None), dict(stats=ODD), dict(k=2, tl=None), dict(k=2, ti=None),
               dict(ws=ODD)):
        assert fwd(**kw) == BAD, kw
    # few rows over several workgroups each
    assert fwd(V=100000, ld=100000, n=8) == SMALL and fwd(V=100000, ld=100000, k=5, ws=None) == SMALL
    assert fwd(N=0, logits=None, tokens=None, lp=None, h=None, stats=None, tl=None, ti=None, k=3) == _lib.CCE_OK

    def bwd(g=P, h=P, logits=P, ld=100, tokens=P, stats=P, N=4, T=1.0, dx=ctypes.c_void_p(8192), ldg=100):
        return lib.cce_token_logprobs_backward(g, h, logits, 1, ld, tokens, 1, stats, N, 100, -100, T, dx, ldg, None)
    for kw in (dict(logits=None), dict(ld=99), dict(tokens=None), dict(stats=None), dict(stats=ODD), dict(T=1e4),
               dict(dx=None), dict(dx=P), dict(ldg=99)):
        assert bwd(**kw) == BAD, kw
    assert bwd(N=0, g=None, h=None, logits=None, tokens=None, stats=None, dx=None) == _lib.CCE_OK


def test_c_linear_token_logprobs(lib):
    def fwd(h=P, w=P, tokens=P, N=4, d=64, V=100, T=1.0, k=0, lp=P, stats=P, tl=P, ti=P, ws=P, n=BIG):
        return lib.cce_linear_token_logprobs_forward(h, w, None, tokens, 1, N, d, V, -100, T, k, lp, P, stats, tl, ti, ws, n,
                                                     None)
    for kw in (dict(h=None), dict(w=None), dict(h=ODD), dict(w=ODD), dict(tokens=None), dict(N=-1), dict(d=60), dict(V=0),
               dict(V=1 << 31), dict(T=0.0), dict(k=101), dict(k=2, ti=None), dict(lp=None), dict(stats=ODD), dict(ws=ODD)):
        assert fwd(**kw) == BAD, kw
    assert fwd(n=8) == SMALL and fwd(k=3, n=4096) == SMALL and fwd(ws=None, n=0) == SMALL
    assert fwd(N=0, h=None, w=None, tokens=None, lp=None, stats=None, ws=None, n=0) == _lib.CCE_OK

    def bwd(h=P, w=P, tokens=P, stats=P, N=4, d=64, V=100, T=1.0, dh=P, dw=P, db=None, ws=P, n=BIG, hdt=0):
        return lib.cce_linear_token_logprobs_backward(P, None, h, w, None, tokens, 1, stats, N, d, V, -100, T, 8192, dh, hdt,
                                                      dw, 0, db, ws, n, None)
    for kw in (dict(h=None), dict(w=None), dict(tokens=None), dict(stats=None), dict(stats=ODD), dict(d=60), dict(V=0),
               dict(V=1 << 33), dict(T=0.0), dict(dh=ODD), dict(hdt=2), dict(db=P)):
        assert bwd(**kw) == BAD, kw
    assert bwd(n=8) == SMALL and bwd(ws=None) == SMALL
    assert bwd(N=0, h=None, w=None, tokens=None, stats=None, dh=None, dw=None) == _lib.CCE_OK


def test_c_rms_norm(lib):
    def fwd(x=P, dt=0, ldx=64, r=P, rdt=0, ldr=64, wdt=0, N=4, D=64, eps=1e-6, y=P, s=P, rstd=P):
        return lib.cce_rms_norm_forward(x, dt, ldx, r, rdt, ldr, P, wdt, N, D, eps, y, s, rstd, None)

    def quant(x=P, dt=0, ldx=64, r=P, rdt=0, ldr=64, wdt=0, N=4, D=64, eps=1e-6, y=P, s=P, rstd=P, qdt=3, group=0):
        return lib.cce_rms_norm_quantized(x, dt, ldx, r, rdt, ldr, P, wdt, N, D, eps, qdt, group, y, rstd, s, None)
    for kw in (dict(x=None), dict(dt=3), dict(ldx=63), dict(rdt=2), dict(dt=1, wdt=1, rdt=0), dict(ldr=63), dict(wdt=2),
               dict(N=-1), dict(D=0), dict(D=(1 << 20) + 1), dict(eps=-1.0), dict(eps=float("nan")), dict(y=None),
               dict(s=None), dict(rstd=None)):
        assert fwd(**kw) == BAD, kw
        assert quant(**kw) == BAD, kw
    for kw in (dict(qdt=0), dict(qdt=5), dict(group=1), dict(group=16), dict(group=96), dict(group=512), dict(group=-32)):
        assert quant(**kw) == BAD, kw
    assert fwd(N=0, x=None, y=None, s=None, rstd=None) == quant(N=0, x=None, y=None, s=None, rstd=None) == _lib.CCE_OK

    def bwd(dy=P, ds=P, s=P, dt=0, sdt=0, ld=64, wdt=0, rstd=P, N=4, D=64, dw=P, ws=P, n=BIG):
        return lib.cce_rms_norm_backward(dy, ds, s, dt, sdt, ld, P, wdt, rstd, N, D, P, None, dw, ws, n, None)
    for kw in (dict(dy=None), dict(s=None), dict(rstd=None), dict(dt=3), dict(sdt=2), dict(ld=63), dict(wdt=2), dict(ws=ODD)):
        assert bwd(**kw) == BAD, kw
    assert bwd(n=8) == SMALL and bwd(ws=None) == SMALL


def test_c_workspaces(lib):
    def size(fn, *args):
        out = ctypes.c_size_t(0)
        assert fn(*args, ctypes.byref(out)) == 0, lib.cce_last_error()
        return out.value
    # nothing for many rows; the splits' sums and candidates for few
    assert size(lib.cce_token_logprobs_workspace_bytes, 4096, 151936, 0) == 0
    assert size(lib.cce_token_logprobs_workspace_bytes, 4096, 151936, 64) == 0
    assert 0 < size(lib.cce_token_logprobs_workspace_bytes, 3, 151936, 0) <= 3 * 64 * 16
    assert 0 < size(lib.cce_token_logprobs_workspace_bytes, 3, 151936, 64) <= 3 * 2048 * 8 + 3 * 128 * 16 + 512
    # beside the cross-entropy's forward: a third sum per split
    ce = _lib.forward_workspace_bytes(4096, 896, 151936, 0, 1)
    assert ce < size(lib.cce_linear_token_logprobs_workspace_bytes, 4096, 896, 151936, 0) <= 2 * ce
    # with alternatives a block of logits, whatever the rows
    for n in (300, 4096, 1 << 20):
        top = size(lib.cce_linear_token_logprobs_workspace_bytes, n, 64, 151936, 20)
        assert top <= (512 << 20) + _lib.forward_workspace_bytes(n, 64, 151936, 0, 1) + (4 << 20)
    # beside the cross-entropy's backward: one number
    ce = _lib.backward_workspace_bytes(4096, 896, 151936, 8192, True, True)
    assert 0 <= size(lib.cce_linear_token_logprobs_backward_workspace_bytes, 4096, 896, 151936, 8192, 1, 0, 1, 0) - ce <= 512
    assert size(lib.cce_rms_norm_backward_workspace_bytes, 1 << 20, 4096, 0, 0) == 0
    assert size(lib.cce_rms_norm_backward_workspace_bytes, 1 << 20, 4096, 0, 1) == 512 * 4096 * 4
    assert size(lib.cce_rms_norm_backward_workspace_bytes, 1 << 20, 1 << 20, 0, 1) <= (64 << 20) + 1024


@pytest.mark.parametrize("V", [100000, 5000, 300000])
@pytest.mark.parametrize("k", [1, 33, 256])
def test_c_blocks_of_logits_have_room(lib, V, k):
    """A last block of few rows is split over more workgroups than a whole one: the workspace holds both."""
    out = ctypes.c_size_t(0)

    def size(n):
        assert lib.cce_linear_token_logprobs_workspace_bytes(n, 72, V, k, ctypes.byref(out)) == 0
        return out.value
    block = max((512 << 20) // (4 * -(-V // 64) * 64) // 256 * 256, 256)

    def rows(n):
        assert lib.cce_token_logprobs_workspace_bytes(n, V, k, ctypes.byref(out)) == 0
        return out.value
    logits = block * 4 * (-(-V // 64) * 64)
    for last in (1, 3, 100, block - 1):
        assert size(block + last) >= logits + max(rows(block), rows(last))
