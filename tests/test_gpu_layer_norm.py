"""Layer norm, forward and backward, against 64-bit references."""
import pytest
import torch

from tests.distill_common import DTYPES, close, half_step

pytestmark = pytest.mark.gpu


def reference(x, w, b, dy, eps):
    """y, dx, dw, db in 64 bits, and sums of the magnitudes that the last three are made of."""
    x, dy = x.double(), dy.double()
    w = torch.ones(x.shape[1]).double() if w is None else w.double()
    mean = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    n = (x - mean) * r
    y = n * w + (0.0 if b is None else b.double())
    a = dy * w
    dx = r * (a - a.mean(1, keepdim=True) - n * (a * n).mean(1, keepdim=True))
    mag = r * (a.abs() + a.abs().mean(1, keepdim=True) + n.abs() * (a * n).abs().mean(1, keepdim=True))
    # the mean is off by a few 2^-24 of the largest |x| (sums of up to D terms in
    # a tree or in runs of D / 256), and so is every difference from it
    shift = (x.abs().amax(1, keepdim=True) + (x - mean).abs()) * r
    return y, dx, (dy * n).sum(0), dy.sum(0), n, mag, shift, (dy * n).abs().sum(0), dy.abs().sum(0), r, a, w


def check(gpu, x, w, b, eps=1e-5, on=None, seed=0):
    from chronicals_amd.kernels.layer_norm import layer_norm
    N, D = x.shape
    dy = torch.randn(N, D, generator=torch.Generator().manual_seed(seed)).to(x.dtype)
    y, dx, dw, db, n, mag, shift, mag_w, mag_b, r, a, w64 = reference(x, w, b, dy, eps)
    xg = (x.to(gpu) if on is None else on).requires_grad_(True)
    wg, bg = (None if p is None else p.to(gpu).requires_grad_(True) for p in (w, b))
    got = layer_norm(xg, wg, bg, eps)
    assert got.dtype == x.dtype and got.shape == x.shape
    # a sum of D terms by 256 threads and a tree: D / 256 + 16 roundings at most;
    # a wave or a workgroup of more threads takes fewer
    e = (D / 256 + 32) * 2.0 ** -24
    rel, least = half_step(x.dtype)
    n_off = e * (shift + 4 * n.abs())
    close(got, y, rel * y.abs() + n_off * w64.abs() + 4 * 2.0 ** -24 * y.abs() + least, "y")
    leaves = [xg] + [p for p in (wg, bg) if p is not None]
    grads = list(torch.autograd.grad(got, leaves, dy.to(gpu)))
    am, anm = a.abs().mean(1, keepdim=True), (a * n).abs().mean(1, keepdim=True)
    off = r * (n_off * anm + n.abs() * (a.abs() * n_off).mean(1, keepdim=True)) + 8 * e * mag + r * e * am
    close(grads.pop(0), dx, rel * dx.abs() + off + least, "dx")
    rows = (N + 64) * 2.0 ** -24
    for p, want, tol in ((wg, dw, rows * mag_w + (dy.double().abs() * n_off).sum(0)), (bg, db, rows * mag_b)):
        if p is not None:
            prel, pleast = half_step(p.dtype)
            close(grads.pop(0), want, prel * want.abs() * (1 + 2.0 ** -7) + tol * (1 + prel) + pleast, "parameter")


@pytest.mark.parametrize("dtype,wdtype", [("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32"),
                                          ("fp32", "fp32")])
@pytest.mark.parametrize("N,D", [(1, 1), (3, 2), (5, 7), (2, 64), (33, 100), (257, 768), (70, 896), (9, 1001), (4, 4096),
                                 (3, 5000), (2, 8200), (2, 20000), (1, 33000), (1500, 72)])
def test_sizes_and_types(gpu, N, D, dtype, wdtype):
    g = torch.Generator().manual_seed(N + D)
    x = (torch.randn(N, D, generator=g) * 2 + 0.5).to(DTYPES[dtype])
    w = (1 + 0.3 * torch.randn(D, generator=g)).to(DTYPES[wdtype])
    b = (0.3 * torch.randn(D, generator=g)).to(DTYPES[wdtype])
    check(gpu, x, w, b)


def test_long_rows(gpu):
    """Longer than the registers hold, with fewer parts of the parameters' gradients."""
    g = torch.Generator().manual_seed(40)
    x = torch.randn(90, 300001, generator=g).bfloat16()
    check(gpu, x, (1 + 0.3 * torch.randn(300001, generator=g)).bfloat16(), None)


@pytest.mark.parametrize("D", [96, 1001, 4096])
def test_without_parameters(gpu, D):
    g = torch.Generator().manual_seed(D)
    x = torch.randn(20, D, generator=g).bfloat16()
    w = (1 + 0.3 * torch.randn(D, generator=g)).bfloat16()
    check(gpu, x, None, None)
    check(gpu, x, w, None)
    check(gpu, x, None, w)


def test_rows_without_variance_and_with_a_large_mean(gpu):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 1024, generator=g)
    x[0] = 0.0
    x[1] = 1.0  # a power of two: the mean is exact
    x[2] += 1000.0
    x[3] *= 1e-4
    x[4, 0] = 1e4
    check(gpu, x, torch.ones(1024), torch.zeros(1024))


def test_strided_rows_and_shapes(gpu):
    from chronicals_amd.kernels.layer_norm import layer_norm
    g = torch.Generator().manual_seed(2)
    big = torch.randn(8, 1030, generator=g)
    w, b = torch.randn(1024, generator=g), torch.randn(1024, generator=g)
    for lo in (0, 1, 4):
        check(gpu, big[:, lo:lo + 1024], w, b, on=big.to(gpu)[:, lo:lo + 1024])
    check(gpu, big[:, :1024], w, b, on=big[:, :1024].t().contiguous().to(gpu).t())
    x = big[:, :1024].to(gpu)
    flat = layer_norm(x, w.to(gpu), b.to(gpu))
    assert torch.equal(layer_norm(x.reshape(2, 4, 1024), w.to(gpu), b.to(gpu)).view(8, 1024), flat)
    assert torch.equal(layer_norm(x[0], w.to(gpu), b.to(gpu)), flat[0])
    # parameters that are views, at any offset
    wide = torch.randn(2, 1025, generator=g).to(gpu)
    assert torch.equal(layer_norm(x, wide[0, 1:], wide[1, 1:]), layer_norm(x, wide[0, 1:].clone(), wide[1, 1:].clone()))


def test_broadcast_input_and_gradient(gpu):
    from chronicals_amd.kernels.layer_norm import layer_norm
    g = torch.Generator().manual_seed(3)
    row = torch.randn(1, 200, generator=g).to(gpu).requires_grad_(True)
    w = torch.randn(200, generator=g).to(gpu).requires_grad_(True)
    layer_norm(row.expand(5, 200), w).sum().backward()
    leaf, wl = row.detach().cpu().double().requires_grad_(True), w.detach().cpu().double().requires_grad_(True)
    torch.nn.functional.layer_norm(leaf.expand(5, 200), (200,), wl).sum().backward()
    assert (row.grad.cpu() - leaf.grad).abs().max() <= 2.0 ** -18 * w.abs().max().item() * 5
    assert (w.grad.cpu() - wl.grad).abs().max() <= 2.0 ** -18 * 5 * 4


def test_no_rows(gpu):
    from chronicals_amd.kernels.layer_norm import layer_norm
    x = torch.zeros(0, 64, device=gpu, requires_grad=True)
    w = torch.ones(64, device=gpu, requires_grad=True)
    y = layer_norm(x, w)
    dx, dw = torch.autograd.grad(y.sum(), [x, w])
    assert y.shape == dx.shape == (0, 64) and not dw.any()


def test_only_what_is_asked(gpu):
    from chronicals_amd.kernels.layer_norm import layer_norm
    g = torch.Generator().manual_seed(4)
    x = torch.randn(50, 512, generator=g).to(gpu)
    w, b = torch.randn(512, generator=g).to(gpu), torch.randn(512, generator=g).to(gpu)
    full = [v.clone().requires_grad_(True) for v in (x, w, b)]
    want = torch.autograd.grad(layer_norm(*full).square().sum(), full)
    for i in range(3):
        some = [v.clone().requires_grad_(i == j) for j, v in enumerate((x, w, b))]
        (got,) = torch.autograd.grad(layer_norm(*some).square().sum(), some[i])
        assert torch.equal(got, want[i])


def test_nan_stays_in_its_row(gpu):
    from chronicals_amd.kernels.layer_norm import layer_norm
    x = torch.randn(4, 300, generator=torch.Generator().manual_seed(5)).to(gpu)
    y = layer_norm(x)
    x[2, 17] = float("nan")
    z = layer_norm(x)
    assert z[2].isnan().all() and torch.equal(z[[0, 1, 3]], y[[0, 1, 3]])


def test_same_bits_streams_and_graphs(gpu):
    from chronicals_amd.kernels.layer_norm import layer_norm
    g = torch.Generator().manual_seed(6)
    a, b = (torch.randn(700, 896, generator=g).bfloat16().to(gpu) for _ in range(2))
    x = a.clone().requires_grad_(True)
    w = torch.randn(896, generator=g).bfloat16().to(gpu).requires_grad_(True)

    def step():
        y = layer_norm(x, w)
        return [y.detach(), *torch.autograd.grad(y, [x, w], b)]
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(4):
        with torch.no_grad():
            x.copy_(b if turn % 2 else a)
        graph.replay()
        got = [v.clone() for v in out]
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, step())), turn


def test_offsets_past_32_bits(gpu):
    from chronicals_amd.kernels.layer_norm import layer_norm
    N, D = 2_200_000, 1024
    x = torch.zeros(N, D, dtype=torch.bfloat16, device=gpu)
    x[-3:] = torch.randn(3, D, generator=torch.Generator().manual_seed(9)).bfloat16().to(gpu)
    few = x[-3:].clone().requires_grad_(True)
    y = layer_norm(few)
    (want,) = torch.autograd.grad(y, few, few.detach())
    x.requires_grad_(True)
    z = layer_norm(x)
    assert torch.equal(z[-3:], y) and not z[:-3].any()
    (dx,) = torch.autograd.grad(z, x, x.detach())
    assert torch.equal(dx[-3:], want)


def test_grad_modes(gpu):
    from chronicals_amd.kernels.layer_norm import layer_norm
    x = torch.randn(5, 64, generator=torch.Generator().manual_seed(8)).to(gpu).requires_grad_(True)
    want = layer_norm(x)
    with torch.inference_mode():
        assert torch.equal(layer_norm(x), want)
    with torch.no_grad():
        assert not layer_norm(x).requires_grad
    assert not layer_norm(x.detach()).requires_grad
    (dx,) = torch.autograd.grad(want.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), x)


def test_module_is_torchs(gpu):
    from chronicals_amd.kernels.layer_norm import LayerNorm
    for kw in ({}, {"bias": False}, {"elementwise_affine": False}):
        ours, theirs = LayerNorm(320, eps=1e-6, **kw).to(gpu), torch.nn.LayerNorm(320, eps=1e-6, **kw).to(gpu)
        theirs.load_state_dict(ours.state_dict())
        x = torch.randn(9, 320, generator=torch.Generator().manual_seed(7)).to(gpu)
        # both in fp32: a few roundings of values below 8
        assert (ours(x) - theirs(x)).abs().max() <= 64 * 2.0 ** -24 * 8
