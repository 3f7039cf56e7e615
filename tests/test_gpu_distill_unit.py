"""The fused distillation's gradient of the logits is held in bf16: what is the same in every row must not be rounded
the same way in every row."""
import pytest
import torch

pytestmark = pytest.mark.gpu

IGNORE = -100


@pytest.mark.parametrize("reduction", ["sum", "mean", "none"])
@pytest.mark.parametrize("N,T,kd,ce,ignored", [
    (300, 1.0, 0.5, 0.5, 0), (300, 2.0, 0.5, 0.5, 40), (20, 2.0, 0.7, 0.3, 0), (300, 1.0, 1.0, 0.0, 0),
    (700, 3.0, 0.9, 0.0, 0), (1, 1.5, 0.0, 0.7, 0),
])
def test_fixed_share(gpu, N, T, kd, ce, ignored, reduction):
    """All logits are 0, so every row's gradient at its label (without labels: at its only entry) is the same number,
    -share + (kd T + ce) / V times the row's factor, which bf16 holds least well: (1 + 2^-8) 2^e / share."""
    from chronicals_amd.kernels.distillation import linear_distillation_loss
    V, d, at, entry = 65536, 64, 40001, 77
    with_labels = ce != 0.0
    share = ce if with_labels else kd * T
    n = N - ignored
    factor = (1 + 2.0 ** -8) / share
    up = factor * n if reduction == "mean" else factor
    h = torch.zeros(N, d)
    h[:, :32] = 1.0
    w = torch.zeros(V, d)
    w[at, 32:] = 1.0  # meets the zeros of h
    bias = torch.zeros(V)
    t, index = torch.zeros(N, 1), torch.full((N, 1), entry if with_labels else at)
    lab = torch.full((N,), at) if with_labels else None
    if ignored:
        lab[::N // ignored][:ignored] = IGNORE
        assert int((lab != IGNORE).sum()) == n
    leaves = [v.to(gpu).requires_grad_(True) for v in (h, w, bias)]
    loss = linear_distillation_loss(leaves[0], leaves[1], t.to(gpu), index.to(gpu), None if lab is None else lab.to(gpu),
                                    leaves[2], temperature=T, distill_weight=kd, ce_weight=ce, reduction=reduction)
    grad_out = torch.full(loss.shape, up, device=gpu)
    dh, dw, db = (v.double().cpu() for v in torch.autograd.grad(loss, leaves, grad_out))
    # in units that make the share a power of two, (kd T + ce) / V of it is what
    # bf16 cannot hold beside it; factors and sums add fp32 roundings, and where the
    # rows have one factor, unit and share are its products rounded to fp32
    tol = (kd * T + ce) / (V * share) + (N + 16) * 2.0 ** -24
    want = (1 + 2.0 ** -8) * ((kd * T + ce) / (V * share) - 1)
    counts = torch.ones(N, dtype=torch.bool) if lab is None else lab != IGNORE
    assert (dh[counts, 32:] / want - 1).abs().max() <= tol and not dh[~counts].any()
    assert (dw[at, :32] / (n * want) - 1).abs().max() <= tol
    assert abs(db[at] / (n * want) - 1) <= tol


def test_factors_that_differ(gpu):
    """Row factors of unlike sizes, zeros, infinities and NaN among them: each row's gradient of the hidden states is
    its factor times that of a factor of 1, to the roundings of both."""
    from chronicals_amd.kernels.distillation import linear_distillation_loss
    g = torch.Generator().manual_seed(3)
    N, V, d, K = 40, 3000, 64, 8
    h = torch.randn(N, d, generator=g).to(gpu).bfloat16().requires_grad_(True)
    w = (torch.randn(V, d, generator=g) * 0.1).to(gpu).bfloat16()
    t = torch.randn(N, K, generator=g).to(gpu)
    index = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(N)]).to(gpu)
    lab = torch.randint(0, V, (N,), generator=g).to(gpu)
    loss = linear_distillation_loss(h, w, t, index, lab, temperature=2.0, distill_weight=0.6, ce_weight=0.3,
                                    reduction="none")
    up = torch.logspace(-30, 30, N, base=10.0)
    up[3], up[7], up[11] = 0.0, float("inf"), float("nan")
    (one,) = torch.autograd.grad(loss, h, torch.ones(N, device=gpu), retain_graph=True)
    (dh,) = torch.autograd.grad(loss, h, up.to(gpu))
    one, dh, up = one.double().cpu(), dh.double().cpu(), up.double()
    finite = up.isfinite()
    # each gradient is a sum of V products whose one factor is off by 2^-8 at most,
    # and is itself rounded to bf16
    x = (h.detach().double() @ w.double().t()).cpu()
    p2, p1 = torch.softmax(x / 2, 1), torch.softmax(x, 1)
    mag = 1.2 * p2 + 0.3 * p1
    mag.scatter_add_(1, index.cpu(), 1.2 * torch.softmax(t.double().cpu() / 2, 1))
    mag.scatter_add_(1, lab.cpu()[:, None], torch.full((N, 1), 0.3).double())
    tol = 2.0 ** -7 * (mag @ w.double().cpu().abs()) + 2.0 ** -7 * one.abs()
    off = (dh - up[:, None] * one).abs()
    assert (off[finite] <= (tol * up[:, None])[finite] * 1.01).all()
    assert not dh[3].any() and not dh[11].isfinite().any()


@pytest.mark.parametrize("temperature", [1.0, 2.0, 3.0])
@pytest.mark.parametrize("bias", [False, True])
def test_rows_read_in_place(gpu, monkeypatch, temperature, bias):
    """The recompute that reads the hidden rows through their order, in several bands and row blocks, with each form of
    the epilogues."""
    from tests.distill_common import labels, teacher
    from tests.test_gpu_distillation import check_linear, head
    g = torch.Generator().manual_seed(70)
    N, d, V = 600, 64, 1200
    h, w = head(g, N, d, V)
    t, index = teacher(g, N, V, 16, 0.3)
    lab = labels(g, N, V, 0.3)
    monkeypatch.setenv("CHRONICALS_CCE_ROW_GATHER", "1")
    monkeypatch.setenv("CHRONICALS_CCE_G_BUDGET_MB", "1")
    b = torch.randn(V, generator=g) if bias else None
    for ce in (0.0, 0.3):
        for reduction in ("mean", "none"):
            check_linear(gpu, h, w, t, index, lab, b, reduction, chunk_size=512, temperature=temperature,
                         distill_weight=0.7, ce_weight=ce)
