"""Distillation from a teacher's top logits against 64-bit references."""
import math

import pytest
import torch

from tests.distill_common import DTYPES, EXP_ERR, EXP_LEAST, IGNORE, close, half_step, labels, reference, teacher

pytestmark = pytest.mark.gpu


def entry_points():
    from chronicals_amd.kernels import distillation
    return distillation


def check_logits(gpu, x, t, index, lab=None, reduction="mean", **how):
    """Loss and gradient of distillation_loss; x etc. are CPU tensors."""
    dt = x.dtype
    rows, grad, counts, mag_rows, mag = reference(x, t, index, lab, how.get("temperature", 1.0),
                                                  how.get("distill_weight", 1.0), how.get("ce_weight", 0.0))
    n = max(int(counts.sum()), 1)
    xd = x.to(gpu).requires_grad_(True)
    loss = entry_points().distillation_loss(xd, t.to(gpu), index.to(gpu), None if lab is None else lab.to(gpu),
                                            reduction=reduction, **how)
    assert loss.dtype == torch.float32
    up = torch.linspace(0.5, 2.0, x.shape[0], dtype=torch.float64) if reduction == "none" else torch.tensor(1.5).double()
    (dx,) = torch.autograd.grad(loss, xd, up.float().to(gpu))
    assert dx.dtype == dt and dx.shape == x.shape
    scale = up[:, None] if reduction == "none" else (up / n if reduction == "mean" else up)
    want = rows if reduction == "none" else rows.sum() / (n if reduction == "mean" else 1)
    tol = mag_rows if reduction == "none" else mag_rows.sum() / (n if reduction == "mean" else 1)
    # as fp32 holds it: past its range it is infinite
    close(loss, want.float().double(), 2 * EXP_ERR * tol, "loss")
    rel, least = half_step(dt)
    g = grad * scale
    # where the loss is infinite the terms of the loss are; the gradient's are not
    T, kd, ce = how.get("temperature", 1.0), how.get("distill_weight", 1.0), how.get("ce_weight", 0.0)
    least = least + EXP_LEAST * (kd * T + ce) * scale
    close(dx, g, rel * g.abs() + 2 * EXP_ERR * mag * scale + least, "dx")
    return loss, dx


LOGITS = [
    # N, V, K, dtype, T, kd, ce, with labels, share of padding
    (1, 1, 1, "fp32", 1.0, 1.0, 0.0, False, 0.0),
    (3, 2, 2, "bf16", 2.0, 1.0, 0.0, False, 0.5),
    (5, 63, 7, "fp32", 0.5, 0.7, 0.3, True, 0.3),
    (4, 8193, 64, "fp16", 1.0, 0.5, 0.5, True, 0.0),
    (7, 50257, 100, "bf16", 4.0, 1.0, 0.0, False, 0.3),
    (2, 50257, 256, "fp32", 1.5, 0.9, 0.1, True, 0.1),
    (1, 20011, 65, "bf16", 100.0, 1.0, 0.0, True, 0.0),
    (1100, 257, 33, "bf16", 2.0, 0.5, 0.5, True, 0.2),
    (9, 1000, 10, "fp32", 1.0, 0.0, 1.0, True, 0.0),
]


@pytest.mark.parametrize("N,V,K,dtype,T,kd,ce,with_labels,pad", LOGITS)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_logits(gpu, N, V, K, dtype, T, kd, ce, with_labels, pad, reduction):
    g = torch.Generator().manual_seed(N * 7 + V)
    x = (torch.randn(N, V, generator=g) * 3).to(DTYPES[dtype])
    t, index = teacher(g, N, V, K, pad, DTYPES[dtype])
    lab = labels(g, N, V) if with_labels else None
    check_logits(gpu, x, t, index, lab, reduction, temperature=T, distill_weight=kd, ce_weight=ce)


def test_logits_sum_int32_and_other_teacher_type(gpu):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 999, generator=g)
    t, index = teacher(g, 6, 999, 20, 0.2, torch.float16, torch.int32)
    check_logits(gpu, x, t, index, labels(g, 6, 999).int(), "sum", temperature=2.0, distill_weight=0.5, ce_weight=0.5)


def test_logits_entries_at_their_edges(gpu):
    """Entries that share a column, a label among them, columns and labels out of range, logits of -inf."""
    g = torch.Generator().manual_seed(2)
    V, K = 5000, 12
    x = torch.randn(8, V, generator=g)
    t, index = teacher(g, 8, V, K)
    index[0] = 17                       # one column
    index[1, ::2] = index[1, 1]
    index[2] = torch.tensor([-1, V, V - 1, 0, 2 ** 40, -2 ** 40, 5, 5, -100, 6, 7, 8])
    t[3, :5] = -math.inf
    t[4] = -math.inf                    # nothing left
    t[5] = torch.finfo(torch.float32).min
    t[6, 0] = torch.finfo(torch.float32).max
    lab = torch.tensor([17, int(index[1, 1]), V - 1, V, -1, 3, int(index[6, 0]), IGNORE])
    for T in (1.0, 0.01, 3.0):
        check_logits(gpu, x, t, index, lab, "none", temperature=T, distill_weight=0.6, ce_weight=0.4)
        check_logits(gpu, x, t, index, None, "mean", temperature=T)


def test_logits_masked_columns_and_rows(gpu):
    """Student logits at -inf and at the type's lowest value, alone and over whole rows; what does not count holds NaN."""
    for dtype in ("bf16", "fp32"):
        dt = DTYPES[dtype]
        low = torch.finfo(dt).min
        g = torch.Generator().manual_seed(3)
        V = 9000
        x = torch.randn(7, V, generator=g).to(dt)
        t, index = teacher(g, 7, V, 10)
        x[0, ::2] = -math.inf
        index[0] = index[0] // 2 * 2 + 1   # the teacher's columns stay
        index[0].clamp_(max=V - 1)
        x[1, ::3] = low
        x[2] = low                         # a uniform row
        x[3, int(index[3, 0])] = -math.inf  # an infinite loss, a finite gradient
        x[4] = math.nan
        x[5, 0] = torch.finfo(dt).max
        x[6] = math.nan
        lab = torch.tensor([1, 4, 3, 2, IGNORE, 0, IGNORE])
        check_logits(gpu, x, t, index, lab, "none", temperature=2.0)
        x[5, 0] = 1.0
        check_logits(gpu, x, t, index, lab, "none", temperature=2.0, distill_weight=0.5, ce_weight=0.5)


def test_logits_nothing_counts(gpu):
    x = torch.full((3, 100), math.nan, device=gpu, requires_grad=True)
    t, index = torch.zeros(3, 4, device=gpu), torch.full((3, 4), -1, device=gpu)
    for lab, kw in ((None, {}), (torch.full((3,), IGNORE, device=gpu), dict(ce_weight=1.0))):
        loss = entry_points().distillation_loss(x, t, index, lab, **kw)
        (dx,) = torch.autograd.grad(loss, x)
        assert loss.item() == 0.0 and not dx.any()


def test_empty_batch(gpu):
    d = entry_points()
    t, index = torch.zeros(0, 4, device=gpu), torch.zeros(0, 4, device=gpu, dtype=torch.int64)
    x = torch.zeros(0, 100, device=gpu, requires_grad=True)
    h = torch.zeros(0, 64, device=gpu, dtype=torch.bfloat16, requires_grad=True)
    w = torch.zeros(100, 64, device=gpu, dtype=torch.bfloat16, requires_grad=True)
    for red in ("mean", "sum", "none"):
        a = d.distillation_loss(x, t, index, reduction=red)
        b = d.linear_distillation_loss(h, w, t, index, reduction=red)
        assert a.shape == b.shape == ((0,) if red == "none" else ())
        if red != "none":
            assert a.item() == b.item() == 0.0
        grads = torch.autograd.grad([a.sum(), b.sum()], [x, h, w])
        assert grads[0].shape == x.shape and grads[1].shape == h.shape and not grads[2].any()


def test_logits_strided(gpu):
    """Padded rows, a transposed tensor, a broadcast one, three dimensions."""
    g = torch.Generator().manual_seed(4)
    V = 3001
    big = torch.randn(6, V + 7, generator=g)
    t, index = teacher(g, 6, V, 8)
    want, grad, _, mag_rows, mag = reference(big[:, 1:V + 1], t, index)
    for x in (big.to(gpu)[:, 1:V + 1], big[:, 1:V + 1].t().contiguous().to(gpu).t()):
        x.requires_grad_(True)
        loss = entry_points().distillation_loss(x.view(2, 3, V) if x.stride(1) == 1 else x, *(
            v.to(gpu).view(2, 3, -1) if x.stride(1) == 1 else v.to(gpu) for v in (t, index)), reduction="none")
        close(loss.reshape(-1), want, 2 * EXP_ERR * mag_rows)
        (dx,) = torch.autograd.grad(loss.sum(), x)
        close(dx, grad, 2.0 ** -23 * grad.abs() + 2 * EXP_ERR * mag)
    one = big[:1, :V].to(gpu).requires_grad_(True)
    loss = entry_points().distillation_loss(one.expand(6, V), t.to(gpu), index.to(gpu), reduction="sum")
    (dx,) = torch.autograd.grad(loss, one)
    _, grad, _, _, mag = reference(big[:1, :V].expand(6, V), t, index)
    close(dx, grad.sum(0, keepdim=True), (2.0 ** -20 + 2 * EXP_ERR) * mag.sum(0, keepdim=True))


def test_logits_gradient_by_differences(gpu):
    """The gradient along a direction against central differences of the loss: these are off by h^2 / 6 of the third
    derivative (below 1 for these losses) and the losses' own error over h."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(4, 300, generator=g).to(gpu)
    t, index = (v.to(gpu) for v in teacher(g, 4, 300, 9, 0.2))
    lab = labels(g, 4, 300, 0.0).to(gpu)
    v = torch.randn(4, 300, generator=g).to(gpu)
    v /= v.norm()
    kw = dict(temperature=2.0, distill_weight=0.5, ce_weight=0.5)
    f = entry_points().distillation_loss
    x.requires_grad_(True)
    (dx,) = torch.autograd.grad(f(x, t, index, lab, **kw), x)
    with torch.no_grad():
        h = 2.0 ** -5
        diff = (f(x + h * v, t, index, lab, **kw).double() - f(x - h * v, t, index, lab, **kw).double()) / (2 * h)
        tol = h * h / 6 + 2 * EXP_ERR * f(x, t, index, lab, **kw).item() / h
    assert abs(diff.item() - (dx * v).sum().item()) <= tol


# ---------------------------------------------------------------------------
# fused with the head's product
# ---------------------------------------------------------------------------

def check_linear(gpu, h, w, t, index, lab=None, bias=None, reduction="mean", frozen=False, chunk_size=8192, **how):
    """h, w bf16 (or of another type whose values bf16 holds), CPU."""
    T, kd, ce = how.get("temperature", 1.0), how.get("distill_weight", 1.0), how.get("ce_weight", 0.0)
    hd, wd = h.double(), w.double()
    x = hd @ wd.t() + (0.0 if bias is None else bias.double())
    rows, grad, counts, mag_rows, mag = reference(x, t, index, lab, T, kd, ce)
    n = max(int(counts.sum()), 1)
    # fp32 accumulation of d products: each logit is off by at most delta
    delta = float((h.shape[1] + 2) * 2.0 ** -24 * (hd.abs() @ wd.abs().t()).max()) + 2.0 ** -24 * float(x.abs().max())
    hg = h.to(gpu).requires_grad_(True)
    wg = w.to(gpu).requires_grad_(not frozen)
    bg = None if bias is None else bias.to(gpu).requires_grad_(True)
    loss = entry_points().linear_distillation_loss(
        hg, wg, t.to(gpu), index.to(gpu), None if lab is None else lab.to(gpu), bg, chunk_size, reduction=reduction,
        **how)
    up = torch.linspace(0.5, 2.0, h.shape[0], dtype=torch.float64) if reduction == "none" else torch.tensor(1.5).double()
    leaves = [hg] + ([] if frozen else [wg]) + ([] if bias is None else [bg])
    grads = torch.autograd.grad(loss, leaves, up.float().to(gpu))
    scale = up[:, None] if reduction == "none" else (up / n if reduction == "mean" else up)
    per_row = 2 * EXP_ERR * mag_rows + 2 * delta * (abs(kd) * T + abs(ce)) * counts
    if reduction == "none":
        close(loss, rows, per_row, "loss")
    else:
        m = n if reduction == "mean" else 1
        close(loss, rows.sum() / m, per_row.sum() / m, "loss")
    # the gradient of the logits G is off by half a step of bf16, by the
    # exponentials and by the logits' own error; products add fp32 rounding
    G, M = grad * scale, mag * scale
    off = 2.0 ** -8 * G.abs() + (2 * EXP_ERR + 2 * delta * max(1.0, 1 / T)) * M
    acc = (max(h.shape[0], w.shape[0]) + 64) * 2.0 ** -24
    wants = [(hg, G @ wd, (off + acc * M) @ wd.abs())]
    if not frozen:
        wants.append((wg, G.t() @ hd, (off + acc * M).t() @ hd.abs()))
    if bias is not None:
        wants.append((bg, G.sum(0), (off + acc * M).sum(0)))
    for got, (leaf, want, tol) in zip(grads, wants):
        assert got.dtype == leaf.dtype and got.shape == leaf.shape
        rel, least = half_step(leaf.dtype)
        close(got, want, rel * want.abs() * (1 + 2.0 ** -7) + tol * (1 + rel) + least, f"gradient {tuple(leaf.shape)}")


def head(g, N, d, V):
    return torch.randn(N, d, generator=g).bfloat16(), (torch.randn(V, d, generator=g) * 0.1).bfloat16()


LINEAR = [
    # N, d, V, K, T, kd, ce, labels, padding, bias, frozen, chunk
    (1, 8, 1, 1, 1.0, 1.0, 0.0, False, 0.0, False, False, 8192),
    (1, 64, 300, 5, 2.0, 1.0, 0.0, False, 0.0, False, False, 8192),
    (17, 72, 1000, 20, 1.0, 0.6, 0.4, True, 0.2, True, False, 256),
    (64, 128, 5003, 64, 2.0, 0.5, 0.5, True, 0.2, False, False, 1024),
    (255, 64, 777, 256, 4.0, 1.0, 0.0, False, 0.3, False, True, 8192),
    (300, 192, 2049, 33, 3.0, 0.5, 0.5, True, 0.2, True, False, 512),
    (300, 1000, 600, 10, 1.0, 1.0, 0.0, True, 0.0, False, False, 8192),
    (700, 64, 1500, 12, 1.5, 0.9, 0.1, True, 0.3, False, True, 512),
]


@pytest.mark.parametrize("N,d,V,K,T,kd,ce,with_labels,pad,bias,frozen,chunk", LINEAR)
def test_linear(gpu, N, d, V, K, T, kd, ce, with_labels, pad, bias, frozen, chunk):
    g = torch.Generator().manual_seed(N + d + V)
    h, w = head(g, N, d, V)
    t, index = teacher(g, N, V, K, pad)
    lab = labels(g, N, V, 0.4) if with_labels else None
    b = torch.randn(V, generator=g) if bias else None
    check_linear(gpu, h, w, t, index, lab, b, "mean", frozen, chunk, temperature=T, distill_weight=kd, ce_weight=ce)


@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_linear_reductions_and_types(gpu, reduction):
    """fp32 and fp16 operands (of values that bf16 holds), int32 indices and labels."""
    g = torch.Generator().manual_seed(9)
    h, w = head(g, 270, 64, 900)
    t, index = teacher(g, 270, 900, 9, 0.3, torch.bfloat16, torch.int32)
    lab = labels(g, 270, 900).int()
    check_linear(gpu, h.float(), w.float(), t, index, lab, None, reduction, temperature=2.0, distill_weight=0.5,
                 ce_weight=0.5)
    check_linear(gpu, h, w.float(), t, index, None, None, reduction)


def test_linear_rows_in_place_and_row_blocks(gpu, monkeypatch):
    """The rows read through their order, and more than one block of rows per band."""
    g = torch.Generator().manual_seed(10)
    h, w = head(g, 600, 64, 1200)
    t, index = teacher(g, 600, 1200, 16, 0.4)
    lab = labels(g, 600, 1200, 0.3)
    monkeypatch.setenv("CHRONICALS_CCE_ROW_GATHER", "1")
    monkeypatch.setenv("CHRONICALS_CCE_G_BUDGET_MB", "1")
    for how in (dict(temperature=2.0, distill_weight=0.5, ce_weight=0.5), dict(temperature=2.0)):
        check_linear(gpu, h, w, t, index, lab, None, **how)
        check_linear(gpu, h, w, t, index, lab, torch.randn(1200, generator=g), **how)


def test_linear_entries_at_their_edges(gpu):
    g = torch.Generator().manual_seed(11)
    V = 2000
    h, w = head(g, 6, 64, V)
    t, index = teacher(g, 6, V, 8)
    index[0] = 1999
    index[1, 1:4] = index[1, 0]
    index[2] = torch.tensor([-1, V, V + 5, 3, 3, 2 ** 40, 255, 256])
    t[3, 2:] = -math.inf
    t[4] = -math.inf
    lab = torch.tensor([1999, int(index[1, 0]), V, 7, 8, IGNORE])
    for T in (1.0, 2.0, 0.25):
        check_linear(gpu, h, w, t, index, lab, chunk_size=256, temperature=T, distill_weight=0.5, ce_weight=0.5)
        check_linear(gpu, h, w, t, index, None, chunk_size=256, temperature=T)


def test_confident_rows_round_once(gpu):
    """Where the student agrees with a sure teacher p and q nearly cancel: the gradient at the teacher's column is their
    difference, not what is left of two rounded values."""
    V, d, N = 1024, 64, 16
    w = torch.zeros(V, d)
    w[torch.arange(d), torch.arange(d)] = 1.0
    h = torch.zeros(N, d)
    h[torch.arange(N), torch.arange(N)] = 14.0
    t = torch.tensor([[14.0, 0.0]]).expand(N, 2).contiguous()
    index = torch.stack([torch.arange(N), torch.arange(N) + 100], 1)
    check_linear(gpu, h.bfloat16(), w.bfloat16(), t, index, reduction="sum")


def test_linear_agrees_with_logits(gpu):
    """Both forms of the loss, and the cross-entropy alone against cut_cross_entropy."""
    from chronicals_amd.kernels.cut_cross_entropy import cut_cross_entropy
    g = torch.Generator().manual_seed(12)
    h, w = (v.to(gpu) for v in head(g, 500, 256, 3000))
    t, index = (v.to(gpu) for v in teacher(g, 500, 3000, 32, 0.2))
    lab = labels(g, 500, 3000).to(gpu)
    d = entry_points()
    kw = dict(temperature=2.0, distill_weight=0.5, ce_weight=0.5)
    a = d.linear_distillation_loss(h, w, t, index, lab, reduction="none", **kw)
    b = d.distillation_loss(h.float() @ w.float().t(), t, index, lab, reduction="none", **kw)
    # logits of fp32 accumulations of 256 products up to 2^-24 * 258 * sum |h w| apart
    delta = 2 * 258 * 2.0 ** -24 * (h.float().abs() @ w.float().abs().t()).max().item()
    assert (a - b).abs().max().item() <= 2 * delta * 1.5 + 4 * EXP_ERR * b.max().item()
    c = d.linear_distillation_loss(h, w, t, index, lab, distill_weight=0.0, ce_weight=1.0)
    e = cut_cross_entropy(h, w, lab)
    assert abs(c.item() - e.item()) <= 2 * delta + 4 * EXP_ERR * e.item()


# ---------------------------------------------------------------------------
# how they are called
# ---------------------------------------------------------------------------

def calls(gpu, seed=20):
    g = torch.Generator().manual_seed(seed)
    h, w = (v.to(gpu).requires_grad_(True) for v in head(g, 300, 64, 5000))
    x = (torch.randn(300, 5000, generator=g) * 2).to(gpu).requires_grad_(True)
    t, index = (v.to(gpu) for v in teacher(g, 300, 5000, 16, 0.2))
    lab = labels(g, 300, 5000).to(gpu)
    d = entry_points()
    kw = dict(temperature=2.0, distill_weight=0.5, ce_weight=0.5)

    def step():
        a = d.distillation_loss(x, t, index, lab, **kw)
        b = d.linear_distillation_loss(h, w, t, index, lab, **kw)
        return [a.detach(), b.detach(), *torch.autograd.grad([a, b], [x, h, w])]
    return step, [h, w, x, t, index, lab]


def test_same_bits_again(gpu):
    step, _ = calls(gpu)
    first = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))


def test_another_stream(gpu):
    step, _ = calls(gpu)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


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


def test_offsets_past_32_bits(gpu):
    """Rows, and rows of the head's weight, that begin past 2^31 elements."""
    d = entry_points()
    g = torch.Generator().manual_seed(24)
    N, V, K = 15000, 151936, 8
    x = torch.zeros(N, V, dtype=torch.bfloat16, device=gpu)
    last = torch.randn(2, V, generator=g).bfloat16()
    x[-2:] = last.to(gpu)
    t, index = teacher(g, 2, V, K)
    tt, ii = torch.zeros(N, K), torch.full((N, K), -1)
    tt[-2:], ii[-2:] = t, index
    x.requires_grad_(True)
    loss = d.distillation_loss(x, tt.to(gpu), ii.to(gpu), reduction="none")
    rows, grad, _, mag_rows, mag = reference(last, t, index)
    close(loss[-2:], rows, 2 * EXP_ERR * mag_rows)
    (dx,) = torch.autograd.grad(loss.sum(), x)
    close(dx[-2:], grad, 2.0 ** -8 * grad.abs() + 2 * EXP_ERR * mag)
    assert not dx[:-2].any()
    values, indices = d.top_logits(x.detach(), K)
    top = torch.sort(last.float(), dim=1, descending=True, stable=True)
    assert torch.equal(values[-2:].float().cpu(), top.values[:, :K]) and torch.equal(indices[-2:].cpu(), top.indices[:, :K])
    del x, dx, loss, values, indices
    N, dim, V = 3, 16384, 140000
    h = (torch.randn(N, dim, generator=g) / 128).bfloat16().to(gpu).requires_grad_(True)
    w = torch.empty(V, dim, dtype=torch.bfloat16, device=gpu).normal_(generator=torch.Generator(gpu).manual_seed(1))
    t, index = teacher(g, N, V, K)
    index[0, 0], index[1, 1] = V - 1, V - 2
    loss = d.linear_distillation_loss(h, w, t.to(gpu), index.to(gpu), reduction="none")
    (dh,) = torch.autograd.grad(loss.sum(), h)
    logits = torch.cat([h.detach().double() @ w[a:a + 10000].double().t() for a in range(0, V, 10000)], 1).cpu()
    rows, grad, _, mag_rows, mag = reference(logits, t, index)
    # sixteen lanes, or the sixteen products of an MFMA step, share out the sum: 1024
    # additions one after the other and a few more, each off by 2^-24 of the magnitudes
    sums = [(h.detach().double().abs() @ w[a:a + 10000].double().abs().t()).max().item() for a in range(0, V, 10000)]
    delta = 2.0 ** -24 * (16384 / 16 + 16) * max(sums)
    close(loss, rows, 2 * EXP_ERR * mag_rows + 2 * delta)
    want, scale = torch.zeros(N, dim).double(), torch.zeros(N, dim).double()
    for a in range(0, V, 10000):
        part = w[a:a + 10000].double().cpu()
        want += grad[:, a:a + 10000] @ part
        scale += mag[:, a:a + 10000] @ part.abs()
    close(dh, want, 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2 * EXP_ERR + V * 2.0 ** -24) * scale)


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


def test_grad_modes(gpu):
    d = entry_points()
    g = torch.Generator().manual_seed(22)
    x = torch.randn(6, 500, generator=g).to(gpu).requires_grad_(True)
    h, w = (v.to(gpu).requires_grad_(True) for v in head(g, 6, 64, 500))
    t, index = (v.to(gpu) for v in teacher(g, 6, 500, 5))
    for f, leaf in ((lambda: d.distillation_loss(x, t, index), x),
                    (lambda: d.linear_distillation_loss(h, w, t, index), h)):
        want = f()
        with torch.inference_mode():
            assert torch.equal(f(), want)
        with torch.no_grad():
            assert not f().requires_grad
        (g1,) = torch.autograd.grad(want, leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g1.float().sum(), leaf)
    # a teacher that requires grad gets none
    tt = t.clone().requires_grad_(True)
    d.distillation_loss(x, tt, index).backward()
    assert tt.grad is None and x.grad is not None
    # twice through one graph
    loss = d.linear_distillation_loss(h, w, t, index)
    a = torch.autograd.grad(loss, [h, w], retain_graph=True)
    b = torch.autograd.grad(loss, [h, w])
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_one_row_without_a_batch(gpu):
    d = entry_points()
    g = torch.Generator().manual_seed(23)
    x = torch.randn(1, 700, generator=g)
    t, index = teacher(g, 1, 700, 6)
    xd = x[0].to(gpu).requires_grad_(True)
    loss = d.distillation_loss(xd, t[0].to(gpu), index[0].to(gpu), torch.tensor(3, device=gpu), reduction="none",
                               ce_weight=0.5)
    rows, grad, _, mag_rows, mag = reference(x, t, index, torch.tensor([3]), ce=0.5)
    close(loss, rows[0], 2 * EXP_ERR * mag_rows[0])
    (dx,) = torch.autograd.grad(loss, xd)
    close(dx, grad[0], 2.0 ** -24 * grad[0].abs() + 2 * EXP_ERR * mag[0])
    h, w = head(g, 1, 64, 700)
    out = d.linear_distillation_loss(h[0].to(gpu), w.to(gpu), t[0].to(gpu), index[0].to(gpu), reduction="none")
    assert out.shape == ()


def test_distillation_step(gpu):
    """A step as it is trained: a teacher's logits kept as its top ones, the student's final norm, the head and both
    losses; gradients of the norm's input and parameters and of the head against 64-bit autograd."""
    from chronicals_amd.kernels.distillation import LinearDistillationLoss, top_logits
    from chronicals_amd.kernels.layer_norm import LayerNorm
    g = torch.Generator().manual_seed(30)
    B, S, d, V, K = 2, 150, 128, 4000, 32
    full = torch.randn(B, S, V, generator=g).to(gpu) * 3
    values, indices = top_logits(full, K)
    assert values.shape == indices.shape == (B, S, K)
    norm = LayerNorm(d, device=gpu, dtype=torch.bfloat16)
    with torch.no_grad():
        norm.weight.copy_(1 + 0.1 * torch.randn(d, generator=g))
        norm.bias.copy_(0.1 * torch.randn(d, generator=g))
    x = torch.randn(B, S, d, generator=g).bfloat16().to(gpu).requires_grad_(True)
    w = (torch.randn(V, d, generator=g) * 0.1).bfloat16().to(gpu).requires_grad_(True)
    lab = labels(g, B * S, V).view(B, S).to(gpu)
    loss = LinearDistillationLoss(temperature=2.0, distill_weight=0.5, ce_weight=0.5)(norm(x), w, values, indices, lab)
    loss.backward()
    ref = {}
    leaves = [v.detach().cpu().double().requires_grad_(True) for v in (x, norm.weight, norm.bias, w)]
    y = torch.nn.functional.layer_norm(leaves[0], (d,), leaves[1], leaves[2], 1e-5)
    z = (y @ leaves[3].t()).view(-1, V)
    lp = torch.log_softmax(z / 2, 1).gather(1, indices.cpu().view(-1, K))
    lq = torch.log_softmax(values.cpu().double().view(-1, K) / 2, 1)
    keep = (lab.cpu().view(-1) != IGNORE)
    kd = 4 * (lq.exp() * (lq - lp)).sum(1)
    ce = torch.nn.functional.cross_entropy(z, lab.cpu().view(-1), ignore_index=IGNORE, reduction="none")
    ref = (0.5 * (kd * keep).sum() + 0.5 * ce.sum()) / keep.sum()
    ref.backward()
    # y is rounded to bf16 (2^-8 of it), which moves each of the logits, sums of d
    # such products, by 2^-8 |y| |w| at most and much less in the mean
    assert abs(loss.item() - ref.item()) <= 2.0 ** -8 * ref.item()
    for got, want in zip((x.grad, norm.weight.grad, norm.bias.grad, w.grad), leaves):
        got, want = got.cpu().double(), want.grad
        # bf16 roundings of y, of the logits' gradient, of the head's result and of
        # the output: four of 2^-8, in the norm of the whole gradient
        assert (got - want).norm() <= 4 * 2.0 ** -8 * want.norm()
