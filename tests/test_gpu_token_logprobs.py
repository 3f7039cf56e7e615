"""Token log-probabilities, entropies and top alternatives against 64-bit references."""
import math

import pytest
import torch

from tests.distill_common import DTYPES, EXP_ERR, EXP_LEAST, IGNORE, close, half_step
from tests.logprobs_common import Reference, tokens

pytestmark = pytest.mark.gpu


def entry_points():
    from chronicals_amd.kernels import token_logprobs
    return token_logprobs


def ups(N, seed=0):
    g = torch.Generator().manual_seed(1000 + seed)
    return torch.randn(N, generator=g), 0.3 * torch.randn(N, generator=g)


def check_top(out, ref, x, k):
    v, i = ref.top(x, k)
    assert torch.equal(out.top_indices.cpu().reshape(i.shape), i)
    lp = v.clone()
    lp[~torch.isfinite(lp)] = 0.0
    close(out.top_logprobs.reshape(v.shape), v, ref.tol[:, None] * (1 + lp.abs()), "top_logprobs")


def check(gpu, x, tok, T=1.0, k=0, on=None, seed=0):
    """Every output and the gradient over CPU logits x [N, V]; `on`: the same values on the device."""
    N = x.shape[0]
    g, h = ups(N, seed)
    ref = Reference(x, tok, T, g, h)
    xd = (x.to(gpu) if on is None else on).requires_grad_(True)
    out = entry_points().token_logprobs(xd, tok.to(gpu), T, k)
    assert out.logprobs.dtype == out.entropy.dtype == torch.float32
    assert (out.top_logprobs is None) == (out.top_indices is None) == (k == 0)
    close(out.logprobs, ref.logprobs, ref.tol, "logprobs")
    close(out.entropy, ref.entropy, ref.tol, "entropy")
    if k:
        check_top(out, ref, x, k)
        assert not out.top_logprobs.requires_grad
    (dx,) = torch.autograd.grad((out.logprobs, out.entropy), xd, (g.to(gpu), h.to(gpu)))
    assert dx.dtype == x.dtype and dx.shape == x.shape
    rel, least = half_step(x.dtype)
    close(dx, ref.grad, rel * ref.grad.abs() + ref.grad_tol + least, "dx")
    return out, dx


SIZES = [
    # N, V, dtype, T, k
    (1, 1, "fp32", 1.0, 1),
    (3, 2, "bf16", 2.0, 2),
    (5, 63, "fp32", 0.5, 7),
    (2, 300, "bf16", 1.0, 256),
    (4, 8193, "fp16", 1.0, 20),
    (7, 50257, "bf16", 0.7, 5),
    (2, 50257, "fp32", 1.5, 100),
    (1, 20011, "bf16", 100.0, 256),
    (3, 4099, "fp32", 0.01, 3),
    (1100, 257, "bf16", 1.0, 33),
    (2100, 1030, "fp16", 0.9, 1),
    (9, 1000, "bf16", 1000.0, 10),
]


@pytest.mark.parametrize("N,V,dtype,T,k", SIZES)
@pytest.mark.parametrize("top", [False, True])
def test_sizes_and_types(gpu, N, V, dtype, T, k, top):
    g = torch.Generator().manual_seed(N * 7 + V)
    x = (torch.randn(N, V, generator=g) * 3).to(DTYPES[dtype])
    check(gpu, x, tokens(g, N, V), T, k if top else 0)


@pytest.mark.parametrize("k", [0, 4])
def test_peaked_rows(gpu, k):
    """Rows that are sure of their token: a log-probability near 0, an entropy near 0, and both small gradients."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(40, 5000, generator=g)
    tok = torch.randint(0, 5000, (40,), generator=g)
    x[torch.arange(40), tok] += torch.linspace(0, 60, 40)
    check(gpu, x, tok, 1.0, k)
    check(gpu, x.bfloat16(), tok.int(), 0.8, k)


@pytest.mark.parametrize("k", [0, 6])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_masked_columns_and_rows(gpu, dtype, k):
    """Logits at -inf and at the type's lowest value, alone and over whole rows; rows that do not count hold NaN."""
    dt = DTYPES[dtype]
    low = torch.finfo(dt).min
    g = torch.Generator().manual_seed(3)
    V = 9000
    x = torch.randn(10, V, generator=g).to(dt)
    x[0, ::2] = -math.inf
    x[1, ::3] = low
    x[2] = low                       # a uniform row
    x[3] = -math.inf                 # nothing left
    x[4] = math.nan
    x[5] = -math.inf
    x[5, 4321] = -3.0                # one column left: it is sure
    x[6, 17] = -math.inf             # the token's own
    x[7] = math.nan
    x[8, :8990] = low                # ten columns above the mask's value
    x[9] = -math.inf
    tok = torch.tensor([1, 4, 3, 2, IGNORE, 4321, 17, IGNORE, 8995, IGNORE])
    for T in (1.0, 2.0, 0.01):
        check(gpu, x, tok, T, k)
    x[5, 0] = torch.finfo(dt).max    # far above the others
    check(gpu, x, tok, 1.0, k)


@pytest.mark.parametrize("k", [0, 3])
def test_not_finite(gpu, k):
    """A NaN or +inf in a row that counts makes its results NaN and no other row's."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(4, 6000, generator=g).to(gpu)
    x[1, 5000] = math.nan
    x[2, 77] = math.inf
    x.requires_grad_(True)
    tok = torch.tensor([3, 3, 3, 3], device=gpu)
    out = entry_points().token_logprobs(x, tok, 1.0, k)
    (dx,) = torch.autograd.grad(out.logprobs.sum() + out.entropy.sum(), x)
    for v in (out.logprobs, out.entropy, dx.sum(1)):
        assert v.isnan().tolist() == [False, True, True, False]
    if k:
        assert out.top_indices[1, 0] == 5000 and out.top_indices[2, 0] == 77


def test_tokens_out_of_range(gpu):
    """No log-probability and no gradient of it; the entropy as any row's."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(6, 700, generator=g)
    tok = torch.tensor([-1, 700, 2 ** 40, 3, IGNORE, -2 ** 40])
    out, _ = check(gpu, x, tok, 1.0, 5)
    assert out.logprobs[[0, 1, 2, 4, 5]].tolist() == [0.0] * 5 and (out.entropy[[0, 1, 2, 5]] > 0).all()
    out = entry_points().token_logprobs(x.to(gpu), torch.tensor([7] * 6, device=gpu), ignore_index=7)
    assert not out.logprobs.any() and not out.entropy.any()


def test_ties_go_to_the_lowest_column(gpu):
    x = torch.zeros(3, 5000)
    x[1, ::7] = 1.0
    x[2, 4000:4100] = 2.0
    for dt in (torch.bfloat16, torch.float32):
        check(gpu, x.to(dt), torch.tensor([0, 7, 4099]), 1.0, 120)


def test_nothing_counts_and_no_rows(gpu):
    t = entry_points()
    x = torch.full((3, 100), math.nan, device=gpu, requires_grad=True)
    out = t.token_logprobs(x, torch.full((3,), IGNORE, device=gpu), top_k=2)
    (dx,) = torch.autograd.grad(out.logprobs.sum() + out.entropy.sum(), x)
    assert not out.logprobs.any() and not out.entropy.any() and not dx.any()
    assert not out.top_logprobs.any() and (out.top_indices == -1).all()
    for k in (0, 3):
        x = torch.zeros(0, 100, device=gpu, requires_grad=True)
        h = torch.zeros(0, 64, device=gpu, dtype=torch.bfloat16, requires_grad=True)
        w = torch.ones(100, 64, device=gpu, dtype=torch.bfloat16, requires_grad=True)
        b = torch.ones(100, device=gpu, requires_grad=True)
        none = torch.zeros(0, device=gpu, dtype=torch.int64)
        a, c = t.token_logprobs(x, none, top_k=k), t.linear_token_logprobs(h, w, none, b, top_k=k)
        for o in (a, c):
            assert o.logprobs.shape == o.entropy.shape == (0,)
            assert k == 0 or o.top_indices.shape == (0, k)
        grads = torch.autograd.grad(sum(o.logprobs.sum() + o.entropy.sum() for o in (a, c)), [x, h, w, b])
        assert grads[0].shape == x.shape and grads[1].shape == h.shape and not grads[2].any() and not grads[3].any()


def test_strides_and_shapes(gpu):
    """Padded rows, a transposed tensor, a broadcast one, three dimensions, a single row."""
    g = torch.Generator().manual_seed(6)
    V = 3001
    big = torch.randn(6, V + 7, generator=g)
    tok = tokens(g, 6, V)
    x = big[:, 1:V + 1]
    for k in (0, 9):
        flat, dflat = check(gpu, x, tok, 1.0, k, on=big.to(gpu)[:, 1:V + 1])
        check(gpu, x, tok, 1.0, k, on=x.t().contiguous().to(gpu).t())
        up, uh = (v.to(gpu) for v in ups(6))
        xd = x.contiguous().to(gpu).view(2, 3, V).requires_grad_(True)
        out = entry_points().token_logprobs(xd, tok.view(2, 3).to(gpu), 1.0, k)
        assert out.logprobs.shape == out.entropy.shape == (2, 3)
        assert k == 0 or out.top_indices.shape == out.top_logprobs.shape == (2, 3, k)
        assert torch.equal(out.logprobs.view(-1), flat.logprobs) and torch.equal(out.entropy.view(-1), flat.entropy)
        (dx,) = torch.autograd.grad((out.logprobs, out.entropy), xd, (up.view(2, 3), uh.view(2, 3)))
        assert torch.equal(dx.view(6, V), dflat)
    one = big[0, :V].to(gpu).requires_grad_(True)
    out = entry_points().token_logprobs(one, torch.tensor(5, device=gpu), top_k=2)
    assert out.logprobs.shape == () and out.top_indices.shape == (2,)
    ref = Reference(big[:1, :V], torch.tensor([5]), 1.0, torch.ones(1), torch.ones(1))
    (dx,) = torch.autograd.grad(out.logprobs + out.entropy, one)
    close(dx, ref.grad[0], 2.0 ** -24 * ref.grad[0].abs() + ref.grad_tol[0])
    row = big[:1, :V].to(gpu).requires_grad_(True)
    out = entry_points().token_logprobs(row.expand(6, V), torch.arange(6, device=gpu))
    (dx,) = torch.autograd.grad(out.logprobs.sum(), row)
    ref = Reference(big[:1, :V].expand(6, V), torch.arange(6), 1.0, torch.ones(6))
    # six rows' gradients added in fp32
    close(dx, ref.grad.sum(0, keepdim=True), 2.0 ** -20 * ref.mag.sum(0, keepdim=True) + ref.grad_tol.sum(0, keepdim=True))


def test_one_gradient_alone(gpu):
    """Either result may be left out: the same as a gradient of zeros for it."""
    g = torch.Generator().manual_seed(7)
    x = torch.randn(5, 800, generator=g).to(gpu).requires_grad_(True)
    h, w = (v.to(gpu).requires_grad_(True) for v in head(g, 5, 64, 800))
    tok = tokens(g, 5, 800).to(gpu)
    t = entry_points()
    for f, leaves in ((lambda: t.token_logprobs(x, tok), [x]), (lambda: t.linear_token_logprobs(h, w, tok), [h, w])):
        for i in range(2):
            got = torch.autograd.grad(f()[i].sum(), leaves)
            out = f()
            want = torch.autograd.grad(out[i].sum() + 0.0 * out[1 - i].sum(), leaves)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradient_by_differences(gpu):
    """The gradient along a direction against central differences: off by h^2 / 6 of the third derivative of a
    log-probability or an entropy along a direction of length 1 (below 8 for these temperatures) and the results' own
    error over h."""
    g = torch.Generator().manual_seed(8)
    x = torch.randn(4, 300, generator=g).to(gpu)
    tok = tokens(g, 4, 300, 0.0)
    v = torch.randn(4, 300, generator=g).to(gpu)
    v /= v.norm()
    up = torch.randn(2, 4, generator=g).to(gpu)
    up /= up.abs().sum()

    def f(x):
        out = entry_points().token_logprobs(x, tok.to(gpu), 1.3)
        return (up[0] * out.logprobs).sum() + (up[1] * out.entropy).sum()
    x.requires_grad_(True)
    (dx,) = torch.autograd.grad(f(x), x)
    with torch.no_grad():
        h = 2.0 ** -5
        diff = (f(x + h * v).double() - f(x - h * v).double()) / (2 * h)
    ref = Reference(x.detach().cpu(), tok, 1.3)
    tol = 8 * h * h / 6 + 2 * ref.tol.max().item() / h
    assert abs(diff.item() - (dx * v).sum().item()) <= tol


def test_agrees_with_the_cross_entropy(gpu):
    """-logprobs is the loss with reduction 'none', and its gradient the loss's."""
    from chronicals_amd.kernels.cut_cross_entropy import cut_cross_entropy
    g = torch.Generator().manual_seed(9)
    h, w = (v.to(gpu) for v in head(g, 300, 128, 3000))
    tok = tokens(g, 300, 3000).to(gpu)
    lp = entry_points().linear_token_logprobs(h, w, tok).logprobs
    loss = cut_cross_entropy(h, w, tok, reduction="none")
    # both are off by the roundings of the sum of exponentials and of a few operations
    ref = Reference((h.double() @ w.double().t()).cpu(), tok.cpu())
    delta = (128 + 2) * 2.0 ** -24 * (h.double().abs() @ w.double().abs().t()).max().item()
    assert ((lp + loss).abs().cpu() <= 2 * ref.tol + 4 * delta).all()


# ---------------------------------------------------------------------------
# fused with the head's product
# ---------------------------------------------------------------------------

def head(g, N, d, V):
    return torch.randn(N, d, generator=g).bfloat16(), (torch.randn(V, d, generator=g) * 0.1).bfloat16()


def check_linear(gpu, h, w, tok, bias=None, T=1.0, k=0, frozen=False, chunk_size=8192, alike=False):
    """h, w bf16 (or of another type whose values bf16 holds), CPU.  With k the logits have to be exact in fp32."""
    hd, wd = h.double(), w.double()
    x = hd @ wd.t() + (0.0 if bias is None else bias.double())
    N, d = h.shape
    g, gh = ups(N, d)
    if alike:
        g, gh = torch.full_like(g, 1.7 / N), torch.full_like(g, 0.01)
    ref = Reference(x, tok, T, g, gh)
    finite = torch.where(x.isfinite(), x, 0.0)
    # fp32 accumulation of d products: each logit is off by at most delta
    delta = float((d + 2) * 2.0 ** -24 * (hd.abs() @ wd.abs().t()).max()) + 2.0 ** -24 * float(finite.abs().max())
    # sums whose maximum or scale is rounded in fp32, where the temperature is low
    scaled = 2.0 ** -22 * float(finite.abs().max()) / T
    off = 2 * delta / T + scaled
    hg = h.to(gpu).requires_grad_(True)
    wg = w.to(gpu).requires_grad_(not frozen)
    bg = None if bias is None else bias.to(gpu).requires_grad_(True)
    out = entry_points().linear_token_logprobs(hg, wg, tok.to(gpu), bg, chunk_size, T, k)
    close(out.logprobs, ref.logprobs, ref.tol + off, "logprobs")
    close(out.entropy, ref.entropy, ref.tol + off * (1 + ref.entropy), "entropy")
    if k:
        check_top(out, ref, x, k)
    assert (out.logprobs <= 0).all()
    leaves = [hg] + ([] if frozen else [wg]) + ([] if bias is None else [bg])
    grads = torch.autograd.grad((out.logprobs, out.entropy), leaves, (g.to(gpu), gh.to(gpu)))
    # the gradient of the logits G is off by half a step of bf16, by the
    # exponentials and by the logits' own error; products add fp32 rounding
    G, M = ref.grad, ref.mag
    e = 2.0 ** -8 * G.abs() * (1 + 2.0 ** -7) + (2 * EXP_ERR + 2 * off * (1 + ref.entropy[:, None])) * M
    # What is below 2^-126 may be lost: of a power of two, before its coefficient
    # (|g| + |h| (1000 + H)) / T at most (the exponent counts from -1000 up), and of G in
    # its unit, which is below 2.  At a low temperature columns have such gradients
    # alone: 0 came out for -1.1e-39.
    e = e + EXP_LEAST * (((g.abs() + gh.abs() * (1000 + ref.entropy)) / T)[:, None] + 2)
    acc = (max(h.shape[0], w.shape[0]) + 64) * 2.0 ** -24
    wants = [(hg, G @ wd, (e + acc * M) @ wd.abs())]
    if not frozen:
        wants.append((wg, G.t() @ hd, (e + acc * M).t() @ hd.abs()))
    if bias is not None:
        wants.append((bg, G.sum(0), (e + acc * M).sum(0)))
    for got, (leaf, want, tol) in zip(grads, wants):
        assert got.dtype == leaf.dtype and got.shape == leaf.shape
        rel, least = half_step(leaf.dtype)
        close(got, want, rel * want.abs() * (1 + 2.0 ** -7) + tol * (1 + rel) + least, f"gradient {tuple(leaf.shape)}")
    return out, grads


LINEAR = [
    # N, d, V, T, bias, frozen, chunk
    (1, 8, 1, 1.0, False, False, 8192),
    (1, 64, 300, 2.0, False, False, 8192),
    (17, 72, 1000, 1.0, True, False, 256),
    (64, 128, 5003, 0.7, False, False, 1024),
    (255, 64, 777, 4.0, False, True, 8192),
    (300, 192, 2049, 1.0, True, False, 512),
    (300, 1000, 600, 1.0, False, False, 8192),
    (700, 64, 1500, 1.5, False, True, 512),
    (700, 64, 1500, 0.5, True, False, 8192),
    (64, 128, 5003, 0.05, True, False, 8192),
    (9, 64, 32768, 1.0, False, False, 8192),   # one round of half-width tiles, exactly
    (9, 64, 32769, 1.0, True, False, 8192),    # whole tiles
    (20, 72, 33000, 1.0, False, True, 8192),   # dH alone, over many splits
    (300, 128, 12000, 0.8, False, True, 8192),
]


@pytest.mark.parametrize("N,d,V,T,bias,frozen,chunk", LINEAR)
def test_linear(gpu, N, d, V, T, bias, frozen, chunk):
    g = torch.Generator().manual_seed(N + d + V)
    h, w = head(g, N, d, V)
    b = torch.randn(V, generator=g) if bias else None
    check_linear(gpu, h, w, tokens(g, N, V, 0.4), b, T, 0, frozen, chunk)


def exact_head(g, N, d, V, bias=False):
    """Values whose products and sums fp32 holds: equal logits come out equal."""
    h = (torch.randn(N, d, generator=g) * 8).round() / 8
    w = (torch.randn(V, d, generator=g) * 16).round() / 128
    return h.bfloat16(), w.bfloat16(), (torch.randn(V, generator=g) * 16).round() / 16 if bias else None


@pytest.mark.parametrize("N,d,V,T,bias,k", [(1, 8, 1, 1.0, False, 1), (3, 64, 300, 2.0, True, 256), (17, 72, 1003, 1.0, True, 5),
                                            (64, 128, 50257, 0.7, False, 20), (300, 1000, 613, 1.0, True, 8),
                                            (700, 64, 1501, 1.0, False, 33), (530, 64, 1502, 1.5, True, 2)])
def test_linear_top(gpu, N, d, V, T, bias, k):
    g = torch.Generator().manual_seed(N + d + V)
    h, w, b = exact_head(g, N, d, V, bias)
    check_linear(gpu, h, w, tokens(g, N, V, 0.3), b, T, k)


@pytest.mark.parametrize("d", [64, 72])
def test_linear_top_several_blocks(gpu, d):
    """More rows than a block of logits holds, the last block short; the first results against the logits' own form."""
    g = torch.Generator().manual_seed(d)
    N, V, k = 1100, 300001, 4
    h, w, _ = exact_head(g, N, d, V)
    tok = tokens(g, N, V, 0.1).to(gpu)
    h, w = h.to(gpu), w.to(gpu)
    x = h.float() @ w.float().t()
    t = entry_points()
    got, want = t.linear_token_logprobs(h, w, tok, top_k=k), t.token_logprobs(x, tok, top_k=k)
    assert torch.equal(got.top_indices, want.top_indices)
    # the same logits, summed over the same workgroups or over others
    for a, b in zip(got[:3], want[:3]):
        assert ((a - b).abs() <= (128 + V / 256) * 2.0 ** -22 * (1 + b.abs())).all()
    plain = t.linear_token_logprobs(h, w, tok)
    for a, b in zip(got[:2], plain[:2]):
        assert ((a - b).abs() <= (128 + V / 256) * 2.0 ** -22 * (1 + b.abs())).all()


def test_linear_types_and_int32(gpu):
    """fp32 and fp16 operands (of values that bf16 holds), int32 tokens."""
    g = torch.Generator().manual_seed(9)
    h, w = head(g, 270, 64, 900)
    tok = tokens(g, 270, 900).int()
    check_linear(gpu, h.float(), w.float(), tok, None, 2.0)
    check_linear(gpu, h, w.float(), tok, torch.randn(900, generator=g).bfloat16().float(), 1.0)
    check_linear(gpu, h.half(), w.half(), tok)


def test_linear_rows_in_place_and_row_blocks(gpu, monkeypatch):
    """The rows read through their order, and more than one block of rows per band."""
    g = torch.Generator().manual_seed(10)
    h, w, b = exact_head(g, 600, 64, 1200, True)
    tok = tokens(g, 600, 1200, 0.3)
    monkeypatch.setenv("CHRONICALS_CCE_ROW_GATHER", "1")
    monkeypatch.setenv("CHRONICALS_CCE_G_BUDGET_MB", "1")
    for k in (0, 3):
        check_linear(gpu, h, w, tok, None, 1.0, k)
        check_linear(gpu, h, w, tok, b, 2.0, k)


@pytest.mark.parametrize("k", [0, 3])
def test_linear_tokens_at_their_edges(gpu, k):
    g = torch.Generator().manual_seed(11)
    V = 2000
    h, w, _ = exact_head(g, 8, 64, V)
    tok = torch.tensor([1999, 0, V, -1, 255, 256, IGNORE, 2 ** 40])
    for T in (1.0, 0.25):
        check_linear(gpu, h, w, tok, None, T, k, chunk_size=256)


@pytest.mark.parametrize("k", [0, 3])
def test_linear_masked_columns(gpu, k):
    """A bias of -inf leaves columns without a probability: a padded vocabulary; of all but one, and of all."""
    g = torch.Generator().manual_seed(12)
    V = 1000
    h, w, b = exact_head(g, 20, 64, V, True)
    tok = tokens(g, 20, 990, 0.2)
    b[990:] = -math.inf
    b[::3] = -math.inf
    check_linear(gpu, h, w, tok, b, 1.0, k)
    b[:] = -math.inf
    b[5] = 1.0
    check_linear(gpu, h, w, tok, b, 2.0, k)
    b[5] = -math.inf
    out, grads = check_linear(gpu, h, w, tok, b, 1.0, k)
    assert not any(v.any() for v in grads)


def test_linear_equal_gradients_of_all_rows(gpu):
    """A mean's gradient is the same number in every row: it is held exactly, not rounded alike everywhere."""
    g = torch.Generator().manual_seed(13)
    N, d, V = 2048, 64, 512
    h = torch.ones(N, d).bfloat16()
    w = (torch.randn(V, d, generator=g) * 0.01).bfloat16()
    tok = torch.randint(0, V, (N,), generator=g)
    out, grads = check_linear(gpu, h, w, tok, alike=True)
    gr, gh = torch.full((N,), 1.7 / N), torch.full((N,), 0.01)
    ref = Reference(h.double() @ w.double().t(), tok, 1.0, gr, gh)
    want = ref.grad.t() @ h.double()
    # rounded alike, the tokens' shares would leave up to 2^-8 of themselves (N / V of
    # them a column); rounded apart, what is left are p's roundings and the output's
    share = 1.7 / N * (tok[:, None] == torch.arange(V)).double().sum(0)[:, None]
    assert ((grads[1].double().cpu() - want).norm() <= 2.0 ** -10 * (share.norm() * math.sqrt(d)) + 2.0 ** -8 * want.norm())


def test_linear_agrees_with_logits(gpu):
    g = torch.Generator().manual_seed(14)
    h, w = (v.to(gpu) for v in head(g, 500, 256, 3000))
    tok = tokens(g, 500, 3000).to(gpu)
    t = entry_points()
    a = t.linear_token_logprobs(h, w, tok, temperature=0.8)
    b = t.token_logprobs(h.float() @ w.float().t(), tok, 0.8)
    # logits of fp32 accumulations of 256 products up to 2^-24 * 258 * sum |h w| apart
    delta = 2 * 258 * 2.0 ** -24 * (h.float().abs() @ w.float().abs().t()).max().item()
    ref = Reference((h.double() @ w.double().t()).cpu(), tok.cpu(), 0.8)
    for x, y in zip(a[:2], b[:2]):
        assert ((x - y).abs().cpu() <= 2 * ref.tol + 2 * delta / 0.8 * (1 + ref.entropy)).all()


# ---------------------------------------------------------------------------
# how they are called
# ---------------------------------------------------------------------------

def calls(gpu, seed=20):
    g = torch.Generator().manual_seed(seed)
    h, w = (v.to(gpu).requires_grad_(True) for v in head(g, 300, 64, 5000))
    x = (torch.randn(300, 5000, generator=g) * 2).to(gpu).requires_grad_(True)
    few = (torch.randn(3, 50000, generator=g) * 2).bfloat16().to(gpu)
    tok = tokens(g, 300, 5000).to(gpu)
    ga, gb = (v.to(gpu) for v in ups(300, seed))
    t = entry_points()

    def step():
        a = t.token_logprobs(x, tok, 0.9, 5)
        b = t.linear_token_logprobs(h, w, tok, temperature=0.9)
        c = t.token_logprobs(few, tok[:3], top_k=40)
        with torch.no_grad():
            d = t.linear_token_logprobs(h, w, tok, top_k=7)
        grads = torch.autograd.grad([a.logprobs, a.entropy, b.logprobs, b.entropy], [x, h, w], [ga, gb, gb, ga])
        return [v.detach() for o in (a, b, c, d) for v in o if v is not None] + list(grads)
    return step, [h, w, x, few, tok, ga, gb]


def test_same_bits_again(gpu):
    step, _ = calls(gpu)
    first = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))


def test_two_streams_at_once(gpu):
    """Calls that overlap on two streams share nothing."""
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
    step, inputs = calls(gpu)
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
    saved = [v.detach().clone() for v in inputs]
    for turn in range(4):
        with torch.no_grad():
            for v, s, o in zip(inputs, saved, other):
                v.copy_(s if turn % 2 else o)
        graph.replay()
        got = [v.clone() for v in out]
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(want, got)), turn


def test_offsets_past_32_bits(gpu):
    """Rows that begin past 2^31 elements."""
    t = entry_points()
    g = torch.Generator().manual_seed(24)
    N, V, k = 15000, 151936, 8
    x = torch.zeros(N, V, dtype=torch.bfloat16, device=gpu)
    last = torch.randn(2, V, generator=g).bfloat16()
    x[-2:] = last.to(gpu)
    tok = torch.full((N,), IGNORE)
    tok[-2:] = torch.tensor([V - 1, 5])
    x.requires_grad_(True)
    a, b = ups(N)
    out = t.token_logprobs(x, tok.to(gpu), top_k=k)
    ref = Reference(last, tok[-2:], 1.0, a[-2:], b[-2:])
    close(out.logprobs[-2:], ref.logprobs, ref.tol)
    close(out.entropy[-2:], ref.entropy, ref.tol)
    v, i = ref.top(last, k)
    assert torch.equal(out.top_indices[-2:].cpu(), i)
    (dx,) = torch.autograd.grad((out.logprobs, out.entropy), x, (a.to(gpu), b.to(gpu)))
    close(dx[-2:], ref.grad, 2.0 ** -8 * ref.grad.abs() + ref.grad_tol + half_step(torch.bfloat16)[1])
    assert not dx[:-2].any()


def test_shared_and_broadcast_leaves(gpu):
    """A head that two calls share, one row for many tokens, a transposed head: each gradient is the sum of the parts'."""
    t = entry_points()
    g = torch.Generator().manual_seed(28)
    h, w = (v.to(gpu) for v in head(g, 12, 64, 2000))
    tok = tokens(g, 12, 2000).to(gpu)
    parts = []
    for rows in (slice(0, 5), slice(5, 12)):
        wl = w.clone().requires_grad_(True)
        t.linear_token_logprobs(h[rows], wl, tok[rows]).logprobs.sum().backward()
        parts.append(wl.grad)
    wl = w.clone().requires_grad_(True)
    sum(t.linear_token_logprobs(h[r], wl, tok[r]).logprobs.sum() for r in (slice(0, 5), slice(5, 12))).backward()
    assert torch.equal(wl.grad, parts[0] + parts[1])

    wt = w.t().contiguous().requires_grad_(True)
    t.linear_token_logprobs(h[:5], wt.t(), tok[:5]).logprobs.sum().backward()
    assert torch.equal(wt.grad.t(), parts[0])

    for f, row in ((lambda x: t.linear_token_logprobs(x, w, tok, top_k=2), h[:1]),
                   (lambda x: t.token_logprobs(x, tok, top_k=2), torch.randn(1, 2000, generator=g).to(gpu))):
        one, many = row.clone().requires_grad_(True), row.repeat(12, 1).requires_grad_(True)
        a, b = f(one.expand(12, -1)), f(many)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        (a.logprobs.sum() + a.entropy.sum()).backward()
        (b.logprobs.sum() + b.entropy.sum()).backward()
        assert torch.equal(one.grad, many.grad.sum(0, keepdim=True))


def test_one_hidden_vector(gpu):
    """Results without a dimension for the rows, and the gradient of a vector."""
    t = entry_points()
    g = torch.Generator().manual_seed(29)
    h, w, _ = exact_head(g, 1, 64, 500)
    x, tok = h.double() @ w.double().t(), torch.tensor([499])
    ref = Reference(x, tok, 1.0, torch.ones(1))
    for k in (0, 3):
        hg = h[0].to(gpu).requires_grad_(True)
        out = t.linear_token_logprobs(hg, w.to(gpu), tok[0].to(gpu), top_k=k)
        assert out.logprobs.shape == out.entropy.shape == ()
        close(out.logprobs, ref.logprobs[0], ref.tol[0])  # the logits are exact
        close(out.entropy, ref.entropy[0], ref.tol[0])
        if k:
            assert out.top_logprobs.shape == (k,) and torch.equal(out.top_indices.cpu(), ref.top(x, k)[1][0])
        out.logprobs.backward()
        # half a step of bf16 of G's elements and of the result; 500 products in fp32
        want, parts = (ref.grad @ w.double())[0], (ref.mag @ w.double().abs())[0]
        err = 2.0 ** -8 * (1 + 2.0 ** -7) * (ref.grad.abs() @ w.double().abs())[0] + (2 * EXP_ERR + 564 * 2.0 ** -24) * parts
        close(hg.grad, want, 2.0 ** -8 * want.abs() * (1 + 2.0 ** -7) + err * (1 + 2.0 ** -8) + half_step(torch.bfloat16)[1])


def test_grad_modes(gpu):
    t = entry_points()
    g = torch.Generator().manual_seed(22)
    x = torch.randn(6, 500, generator=g).to(gpu).requires_grad_(True)
    h, w = (v.to(gpu).requires_grad_(True) for v in head(g, 6, 64, 500))
    tok = tokens(g, 6, 500).to(gpu)
    for f, leaf in ((lambda: t.token_logprobs(x, tok), x), (lambda: t.linear_token_logprobs(h, w, tok), h)):
        want = f()
        with torch.inference_mode():
            assert torch.equal(f().logprobs, want.logprobs)
        with torch.no_grad():
            assert not f().logprobs.requires_grad
        loss = want.logprobs.sum() + want.entropy.square().sum()
        a = torch.autograd.grad(loss, leaf, retain_graph=True)
        b = torch.autograd.grad(loss, leaf, create_graph=True)
        assert torch.equal(a[0], b[0])
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(b[0].float().sum(), leaf)


def test_policy_step(gpu):
    """A step as it is trained: the residual's addition and the final norm, the head, log-probabilities of the answer's
    tokens with an entropy term; gradients against 64-bit autograd."""
    from chronicals_amd.kernels.rms_norm import RMSNorm
    g = torch.Generator().manual_seed(30)
    B, S, d, V = 2, 150, 128, 4000
    norm = RMSNorm(d, device=gpu, dtype=torch.bfloat16)
    with torch.no_grad():
        norm.weight.copy_(1 + 0.1 * torch.randn(d, generator=g))
    x = torch.randn(B, S, d, generator=g).bfloat16().to(gpu).requires_grad_(True)
    r = torch.randn(B, S, d, generator=g).to(gpu).requires_grad_(True)
    w = (torch.randn(V, d, generator=g) * 0.1).bfloat16().to(gpu).requires_grad_(True)
    tok = tokens(g, B * S, V).view(B, S).to(gpu)
    adv = torch.randn(B, S, generator=g).to(gpu)
    n = (tok != IGNORE).sum()
    y, s = norm(x, r)
    out = entry_points().linear_token_logprobs(y, w, tok, temperature=0.9)
    loss = -(adv * out.logprobs).sum() / n - 0.01 * out.entropy.sum() / n + 1e-3 * s.square().mean()
    loss.backward()
    leaves = [v.detach().cpu().double().requires_grad_(True) for v in (x, r, norm.weight, w)]
    sr = leaves[0] + leaves[1]
    yr = sr / torch.sqrt(sr.square().mean(-1, keepdim=True) + 1e-6) * leaves[2]
    lp = torch.log_softmax((yr @ leaves[3].t()).view(-1, V) / 0.9, 1)
    keep = (tok.cpu().view(-1) != IGNORE)
    picked = lp.gather(1, tok.cpu().view(-1, 1).clamp(min=0))[:, 0] * keep
    H = -(lp.exp() * lp).sum(1) * keep
    ref = -(adv.cpu().double().view(-1) * picked).sum() / keep.sum() - 0.01 * H.sum() / keep.sum()
    ref = ref + 1e-3 * sr.square().mean()
    ref.backward()
    for got, want in zip((x.grad, r.grad, norm.weight.grad, w.grad), leaves):
        got, want = got.cpu().double(), want.grad
        # bf16 roundings of y, of the logits' gradient, of the head's result and of
        # the output: four of 2^-8, in the norm of the whole gradient
        assert (got - want).norm() <= 4 * 2.0 ** -8 * want.norm()
