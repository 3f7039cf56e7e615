"""RMS norm with the residual's addition, its gradients and its 8-bit form, against 64-bit references."""
import math

import pytest
import torch

from tests.distill_common import DTYPES, close, half_step

pytestmark = pytest.mark.gpu


def entry_points():
    from chronicals_amd.kernels import rms_norm
    return rms_norm


def e(D):
    """Relative error of a sum of D terms by 256 threads and a tree (more threads, or a wave, take fewer additions), and
    of the few operations behind it."""
    return (D / 256 + 32) * 2.0 ** -24


def summed(x, r):
    """x + r as the residual's type holds it: one rounding of the fp32 sum."""
    return x if r is None else (x.float() + r.float()).to(r.dtype)


def inputs(N, D, dtype, wdtype=None, rdtype=None, seed=0):
    g = torch.Generator().manual_seed(N + D + seed)
    x = (torch.randn(N, D, generator=g) * 2 + 0.5).to(DTYPES[dtype])
    w = (1 + 0.3 * torch.randn(D, generator=g)).to(DTYPES[wdtype]) if wdtype else None
    r = (3 * torch.randn(N, D, generator=g)).to(DTYPES[rdtype]) if rdtype else None
    return x, w, r


def check(gpu, x, w, r, eps=1e-6, on=None, seed=0, with_ds=True):
    """y, s and every gradient; `on`: x and r with the same values on the device."""
    N, D = x.shape
    g = torch.Generator().manual_seed(seed)
    dy = torch.randn(N, D, generator=g).to(x.dtype)
    ds = torch.randn(N, D, generator=g).to(r.dtype) if r is not None and with_ds else None
    s = summed(x, r).double()
    w64 = torch.ones(D).double() if w is None else w.double()
    rstd = 1 / torch.sqrt(s.square().mean(1, keepdim=True) + eps)
    n = s * rstd
    y, a = n * w64, dy.double() * w64
    an = (a * n).mean(1, keepdim=True)
    dx = rstd * (a - n * an) + (0.0 if ds is None else ds.double())
    xg, rg = (x.to(gpu), None if r is None else r.to(gpu)) if on is None else on
    wg = None if w is None else w.to(gpu).requires_grad_(True)
    xg.requires_grad_(True)
    got = entry_points().rms_norm(xg, wg, None if rg is None else rg.requires_grad_(True), eps)
    if r is not None:
        got, sg = got
        assert sg.dtype == r.dtype and torch.equal(sg.cpu(), summed(x, r))
    assert got.dtype == x.dtype and got.shape == x.shape
    rel, least = half_step(x.dtype)
    close(got, y, rel * y.abs() + e(D) * y.abs() + least, "y")
    leaves = [v for v in (xg, rg, wg) if v is not None]
    outs, ups = ([got], [dy.to(gpu)]) if ds is None else ([got, sg], [dy.to(gpu), ds.to(gpu)])
    grads = dict(zip(map(id, leaves), torch.autograd.grad(outs, leaves, ups)))
    mag = rstd * (a.abs() + n.abs() * (a * n).abs().mean(1, keepdim=True)) + (0.0 if ds is None else ds.double().abs())
    for leaf in (xg, rg):
        if leaf is not None:
            assert grads[id(leaf)].dtype == leaf.dtype
            lrel, lleast = half_step(leaf.dtype)
            close(grads[id(leaf)], dx, lrel * dx.abs() + 8 * e(D) * mag + lleast, "dx")
    if w is not None:
        terms = dy.double() * n
        tol = ((N + 64) * 2.0 ** -24 + e(D)) * terms.abs().sum(0)
        prel, pleast = half_step(w.dtype)
        want = terms.sum(0)
        close(grads[id(wg)], want, prel * want.abs() * (1 + 2.0 ** -7) + tol * (1 + prel) + pleast, "dw")


TYPES = [("bf16", "bf16", "bf16"), ("bf16", "fp32", "fp32"), ("bf16", "bf16", None), ("fp16", "fp16", "fp16"),
         ("fp16", "fp32", "fp32"), ("fp16", "fp16", None), ("fp32", "fp32", "fp32"), ("fp32", "fp32", None)]
SIZES = [(1, 1), (3, 2), (5, 7), (2, 64), (33, 100), (257, 768), (70, 896), (9, 1001), (4, 4096), (3, 5000), (2, 8200),
         (2, 20000), (1, 33000), (1500, 72)]


@pytest.mark.parametrize("dtype,wdtype,rdtype", TYPES)
@pytest.mark.parametrize("N,D", SIZES)
def test_sizes_and_types(gpu, N, D, dtype, wdtype, rdtype):
    check(gpu, *inputs(N, D, dtype, wdtype, rdtype))


@pytest.mark.parametrize("D", [96, 1001, 4096, 20000])
def test_without_weight_or_gradient_of_the_sum(gpu, D):
    x, w, r = inputs(20, D, "bf16", "bf16", "bf16")
    check(gpu, x, None, None)
    check(gpu, x, None, r)
    check(gpu, x, w, r, with_ds=False)
    check(gpu, x, w, r.float(), with_ds=False)


def test_long_rows(gpu):
    """Longer than the registers hold, with fewer parts of the weight's gradient."""
    check(gpu, *inputs(90, 300001, "bf16", "bf16", "fp32"))


def test_rows_at_the_edges(gpu):
    """Rows of zeros, of one value, tiny and large ones; eps of 0."""
    x, w, _ = inputs(6, 1024, "fp32", "fp32")
    x[0] = 0.0
    x[1] = 1.0
    x[2] += 1000.0
    x[3] *= 1e-4
    x[4, 0] = 1e4
    check(gpu, x, w, None)
    r = torch.randn(6, 1024, generator=torch.Generator().manual_seed(1))
    r[1] = -x[1]  # a sum of zeros
    check(gpu, x, w, r)
    check(gpu, x[2:], w, r[2:], eps=0.0)


def test_strided_rows_and_shapes(gpu):
    f = entry_points().rms_norm
    g = torch.Generator().manual_seed(2)
    big, res = torch.randn(8, 1030, generator=g), torch.randn(8, 1029, generator=g)
    w = torch.randn(1024, generator=g)
    for lo in (0, 1, 4):
        x, r = big[:, lo:lo + 1024], res[:, 5 - lo:1029 - lo]
        check(gpu, x, w, r, on=(big.to(gpu)[:, lo:lo + 1024], res.to(gpu)[:, 5 - lo:1029 - lo]))
        check(gpu, x, w, None, on=(big.to(gpu)[:, lo:lo + 1024], None))
    x, r = big[:, :1024], res[:, :1024]
    check(gpu, x, w, r, on=tuple(v.t().contiguous().to(gpu).t() for v in (x, r)))
    xg, rg, wg = x.to(gpu), r.to(gpu), w.to(gpu)
    flat = f(xg, wg, rg)
    for a, b in zip(f(xg.reshape(2, 4, 1024), wg, rg.reshape(2, 4, 1024)), flat):
        assert a.shape == (2, 4, 1024) and torch.equal(a.view(8, 1024), b)
    for a, b in zip(f(xg[0], wg, rg[0]), flat):
        assert torch.equal(a, b[0])
    wide = torch.randn(2, 1025, generator=g).to(gpu)
    assert torch.equal(f(xg, wide[0, 1:]), f(xg, wide[0, 1:].clone()))


def test_broadcast_inputs(gpu):
    g = torch.Generator().manual_seed(3)
    row = torch.randn(1, 200, generator=g)
    r = torch.randn(5, 200, generator=g)
    w = torch.randn(200, generator=g)
    rg, wg, lg = (v.to(gpu).requires_grad_(True) for v in (r, w, row))
    y, s = entry_points().rms_norm(lg.expand(5, 200), wg, rg)
    (y.sum() + s.sum()).backward()
    leaves = [v.double().requires_grad_(True) for v in (row, r, w)]
    t = leaves[0].expand(5, 200) + leaves[1]
    (t / torch.sqrt(t.square().mean(1, keepdim=True) + 1e-6) * leaves[2]).sum().add(t.sum()).backward()
    for got, want, n in zip((lg, rg, wg), leaves, (5, 1, 5)):
        # five rows at most, each off by a few 2^-24 of the magnitudes
        assert (got.grad.cpu() - want.grad).abs().max() <= 2.0 ** -18 * n * (2 + w.abs().max().item())


def test_no_rows(gpu):
    x = torch.zeros(0, 64, device=gpu, requires_grad=True)
    r = torch.zeros(0, 64, device=gpu, requires_grad=True)
    w = torch.ones(64, device=gpu, requires_grad=True)
    y, s = entry_points().rms_norm(x, w, r)
    dx, dr, dw = torch.autograd.grad(y.sum() + s.sum(), [x, r, w])
    assert y.shape == s.shape == dx.shape == dr.shape == (0, 64) and not dw.any()
    for group in (None, 32):
        q, scales = entry_points().rms_norm_quantized(x, w, group_size=group)
        assert q.shape == (0, 64) and scales.shape == ((0,) if group is None else (0, 2))


@pytest.mark.parametrize("rdtype", ["bf16", "fp32"])
def test_only_what_is_asked(gpu, rdtype):
    x, w, r = inputs(50, 512, "bf16", "fp32", rdtype)
    leaves = [v.to(gpu) for v in (x, w, r)]

    def loss(a):
        y, s = entry_points().rms_norm(*a)
        return y.float().square().sum() + s.float().square().sum()
    full = [v.clone().requires_grad_(True) for v in leaves]
    want = torch.autograd.grad(loss(full), full)
    for i in range(3):
        some = [v.clone().requires_grad_(i == j) for j, v in enumerate(leaves)]
        (got,) = torch.autograd.grad(loss(some), some[i])
        assert torch.equal(got, want[i])
    # the sum's gradient alone passes through
    y, s = entry_points().rms_norm(*full)
    up = torch.randn_like(s)
    for got, v in zip(torch.autograd.grad(s, [full[0], full[2]], up), (full[0], full[2])):
        assert torch.equal(got, up.to(v.dtype))


def test_gradient_by_differences(gpu):
    """Along a direction, against central differences of a scalar made of both results: off by h^2 / 6 of its third
    derivative (below 200 here: rows of size 1 in 40 dimensions) and the results' own error over h."""
    g = torch.Generator().manual_seed(8)
    x, r, v = (torch.randn(4, 40, generator=g).to(gpu) for _ in range(3))
    w, up, us = (torch.randn(*s, generator=g).to(gpu) for s in ((40,), (4, 40), (4, 40)))
    v /= v.norm()

    def f(x):
        y, s = entry_points().rms_norm(x, w, r)
        return (y.double() * up.double()).sum() + (s.double() * us.double()).sum()
    x.requires_grad_(True)
    (dx,) = torch.autograd.grad(f(x), x)
    with torch.no_grad():
        h = 2.0 ** -7
        diff = (f(x + h * v) - f(x - h * v)) / (2 * h)
        y, s = entry_points().rms_norm(x, w, r)
        off = 2.0 ** -22 * ((y.abs() * up.abs()).sum() + (s.abs() * us.abs()).sum()).item()
    assert abs(diff.item() - (dx.double() * v.double()).sum().item()) <= 200 * h * h / 6 + 2 * off / h


def test_not_finite_stays_in_its_row(gpu):
    f = entry_points()
    x = torch.randn(4, 300, generator=torch.Generator().manual_seed(5)).to(gpu)
    y = f.rms_norm(x)
    q, scales = f.rms_norm_quantized(x, group_size=32)
    x[2, 17] = math.nan
    z = f.rms_norm(x)
    assert torch.equal(z[[0, 1, 3]], y[[0, 1, 3]]) and z[2].isnan().all()
    for dtype in (torch.float8_e4m3fn, torch.int8):
        p, t = f.rms_norm_quantized(x, dtype=dtype, group_size=32)
        assert t[2].isnan().all() and not t[[0, 1, 3]].isnan().any()
        p, t = f.rms_norm_quantized(x, dtype=dtype)
        assert t.isnan().tolist() == [False, False, True, False]
    p, t = f.rms_norm_quantized(x, group_size=32)
    assert torch.equal(p.view(torch.uint8)[[0, 1, 3]], q.view(torch.uint8)[[0, 1, 3]]) and torch.equal(t[3], scales[3])


# ---------------------------------------------------------------------------
# in 8 bits
# ---------------------------------------------------------------------------

MOST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def check_quantized(gpu, x, w, r, dtype, group, on=None, eps=1e-6):
    N, D = x.shape
    s = summed(x, r).double()
    y = s / torch.sqrt(s.square().mean(1, keepdim=True) + eps) * (1.0 if w is None else w.double())
    xg, rg = (x.to(gpu), None if r is None else r.to(gpu)) if on is None else on
    q, scales, *kept = entry_points().rms_norm_quantized(xg, None if w is None else w.to(gpu), rg, eps, dtype, group)
    assert q.dtype == dtype and q.shape == x.shape and scales.dtype == torch.float32
    assert len(kept) == (r is not None) and (r is None or torch.equal(kept[0].cpu(), summed(x, r)))
    size = group or D
    groups = -(-D // size)
    assert scales.shape == ((N,) if group is None else (N, groups))
    padded = torch.zeros(N, groups * size).double()
    padded[:, :D] = y.abs()
    want = padded.view(N, groups, size).amax(2).clamp(min=1e-30) / MOST[dtype]
    # the scale is y's error and two roundings off
    close(scales.view(N, groups), want, (e(D) + 4 * 2.0 ** -24) * want, "scales")
    by = want.repeat_interleave(size, 1)[:, :D]
    v = y / by
    # half a step of the type at v, and the roundings of v before it
    half = torch.full_like(v, 0.5) if dtype == torch.int8 else torch.maximum(
        2.0 ** (torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 4), torch.tensor(2.0 ** -10).double())
    got = q.cpu().double() if dtype == torch.int8 else q.cpu().float().double()
    close(got, v, half * (1 + 2.0 ** -20) + (2 * e(D) + 8 * 2.0 ** -24) * v.abs(), "q")
    return q, scales


@pytest.mark.parametrize("dtype", list(MOST))
@pytest.mark.parametrize("group", [None, 32, 64, 128, 256])
@pytest.mark.parametrize("kind", TYPES)
def test_quantized_groups_and_types(gpu, kind, group, dtype):
    for N, D in ((3, 640), (2, 1001), (2, 9000)):
        check_quantized(gpu, *inputs(N, D, *kind), dtype, group)


@pytest.mark.parametrize("dtype", list(MOST))
@pytest.mark.parametrize("N,D", SIZES)
def test_quantized_sizes(gpu, N, D, dtype):
    x, w, r = inputs(N, D, "bf16", "bf16", "bf16")
    for group in (None, 128):
        check_quantized(gpu, x, w, r, dtype, group)
        check_quantized(gpu, x, None, None, dtype, group)


@pytest.mark.parametrize("dtype", list(MOST))
def test_quantized_rows_at_the_edges(gpu, dtype):
    """Rows and groups of zeros, of one value, of far apart sizes, and what is too small for a scale of its own."""
    x, w, _ = inputs(6, 1024, "fp32", "fp32")
    x[0] = 0.0
    x[1] = 1.0
    x[2, :512] = 0.0
    x[3, ::2] *= 1e-6
    x[4, 0] = 1e4
    x[5, 128:256] *= 1e-35
    for group in (None, 128):
        q, scales = check_quantized(gpu, x, w, None, dtype, group)
        assert not q.view(torch.uint8)[0].any() and (scales > 0).all()


def test_quantized_strides_and_shapes(gpu):
    f = entry_points().rms_norm_quantized
    g = torch.Generator().manual_seed(2)
    big, res = torch.randn(8, 1030, generator=g), torch.randn(8, 1029, generator=g)
    w = torch.randn(1024, generator=g)
    for lo in (0, 1, 4):
        check_quantized(gpu, big[:, lo:lo + 1024], w, res[:, 5 - lo:1029 - lo], torch.float8_e4m3fn, 64,
                        on=(big.to(gpu)[:, lo:lo + 1024], res.to(gpu)[:, 5 - lo:1029 - lo]))
    x, r = big[:, :1024].to(gpu), res[:, :1024].to(gpu)
    flat = f(x, w.to(gpu), r, group_size=128)
    for a, b in zip(f(x.reshape(2, 4, 1024), w.to(gpu), r.reshape(2, 4, 1024), group_size=128), flat):
        assert a.shape[:2] == (2, 4) and torch.equal(a.reshape(b.shape).view(torch.uint8), b.view(torch.uint8))
    q, scales, s = f(x[0], w.to(gpu), r[0])
    assert scales.shape == () and q.shape == s.shape == (1024,)


@pytest.mark.parametrize("group", [None, 256])
@pytest.mark.parametrize("dtype", list(MOST))
def test_quantized_rounds_to_nearest_even(gpu, dtype, group):
    """Every number of the type, every midpoint between two, and the midpoints' neighbours on either side.  A row of
    ones has a mean square of 1, so with eps 0 y is the weight, whose largest value makes the scale 1."""
    codes = torch.arange(0, 0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn).float() if dtype != torch.int8 else \
        torch.arange(0, 128).float()
    mid = (codes[:-1] + codes[1:]) / 2
    v = torch.cat([codes, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20)])
    w = torch.zeros(1024)
    w[:v.numel()], w[512:512 + v.numel()] = v, -v
    w[::256] = MOST[dtype]
    q, scales = entry_points().rms_norm_quantized(torch.ones(1, 1024, device=gpu), w.to(gpu), None, 0.0, dtype, group)
    assert (scales == 1.0).all()
    want = torch.round(w) if dtype == torch.int8 else w.to(dtype).float()
    assert torch.equal(q[0].cpu().float(), want)


# ---------------------------------------------------------------------------
# how they are called
# ---------------------------------------------------------------------------

def calls(gpu, seed=20):
    x, w, r = (v.to(gpu) for v in inputs(300, 896, "bf16", "fp32", "fp32", seed))
    g = torch.Generator().manual_seed(seed)
    dy, ds = torch.randn(300, 896, generator=g).bfloat16().to(gpu), torch.randn(300, 896, generator=g).to(gpu)
    for v in (x, w, r):
        v.requires_grad_(True)
    f = entry_points()

    def step():
        y, s = f.rms_norm(x, w, r)
        q = f.rms_norm_quantized(x, w, r, group_size=128)
        p = f.rms_norm_quantized(x, w, dtype=torch.int8)
        return [y.detach(), s.detach(), *(v.view(torch.uint8) if v.element_size() == 1 else v for v in (*q, *p)),
                *torch.autograd.grad((y, s), [x, w, r], (dy, ds))]
    return step, [x, w, r, dy, ds]


def test_same_bits_again(gpu):
    step, _ = calls(gpu)
    first = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))


def test_two_streams_at_once(gpu):
    steps = [calls(gpu, s)[0] for s in (20, 21)]
    want = [f() for f in steps]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (f, s) in enumerate(zip(steps, streams)):
            with torch.cuda.stream(s):
                got[i].append(f())
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        for r in runs:
            assert all(torch.equal(a, b) for a, b in zip(w, r))


def test_captured_and_replayed(gpu):
    step, inputs_ = calls(gpu)
    other = calls(gpu, 21)[1]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    saved = [v.detach().clone() for v in inputs_]
    for turn in range(4):
        with torch.no_grad():
            for v, s, o in zip(inputs_, saved, other):
                v.copy_(s if turn % 2 else o)
        graph.replay()
        got = [v.clone() for v in out]
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(want, got)), turn


def test_offsets_past_32_bits(gpu):
    """Rows that begin past 2^31 elements."""
    f = entry_points()
    N, D = 600000, 4096
    x = torch.ones(N, D, dtype=torch.bfloat16, device=gpu)
    g = torch.Generator().manual_seed(1)
    last = torch.randn(3, D, generator=g).bfloat16()
    x[-3:] = last.to(gpu)
    w = torch.randn(D, generator=g).bfloat16()
    y = f.rms_norm(x, w.to(gpu))
    s = last.double()
    want = s / torch.sqrt(s.square().mean(1, keepdim=True) + 1e-6) * w.double()
    close(y[-3:], want, (2.0 ** -8 + e(D)) * want.abs())
    del y
    q, scales = f.rms_norm_quantized(x, w.to(gpu), group_size=128)
    p, t = f.rms_norm_quantized(last.to(gpu), w.to(gpu), group_size=128)
    assert torch.equal(q[-3:].view(torch.uint8), p.view(torch.uint8)) and torch.equal(scales[-3:], t)


def test_stream_changed_in_place(gpu):
    """y may be changed in place; a sum that a backward needs may not without its knowledge."""
    x, w, r = (v.to(gpu).requires_grad_(True) for v in inputs(12, 64, "fp32", "fp32", "fp32"))
    f = entry_points().rms_norm
    y, s = f(x, w, r)
    want = torch.autograd.grad(torch.relu(y + 1).sum() + s.sum(), [x, w, r])
    y, s = f(x, w, r)
    y += 1
    y.relu_()
    got = torch.autograd.grad(y.sum() + s.sum(), [x, w, r])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    y, s = f(x, w, r)
    with torch.no_grad():
        s += 1
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


def test_gradients_are_not_differentiated_again(gpu):
    x, w, r = (v.to(gpu).requires_grad_(True) for v in inputs(12, 64, "fp32", "fp32", "fp32"))
    y, s = entry_points().rms_norm(x, w, r)
    loss = y.square().sum() + s.sum()
    plain = torch.autograd.grad(loss, [x, w, r], retain_graph=True)
    again = torch.autograd.grad(loss, [x, w, r], create_graph=True)
    for p, a, leaf in zip(plain, again, (x, w, r)):
        assert torch.equal(p, a)
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(a.square().sum(), leaf, retain_graph=True)


def test_module(gpu):
    from chronicals_amd.kernels.rms_norm import RMSNorm
    norm = RMSNorm(64, device=gpu, dtype=torch.bfloat16)
    assert list(norm.state_dict()) == ["weight"]
    x = torch.randn(3, 5, 64, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)
    assert torch.equal(norm(x), entry_points().rms_norm(x, norm.weight))
    y, s = norm(x, x)
    assert torch.equal(s, x + x) and y.shape == x.shape
