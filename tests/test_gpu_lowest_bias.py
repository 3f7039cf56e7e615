"""Log-probabilities from hidden states where a bias masks columns with its type's lowest value."""
import math

import pytest
import torch

from tests.distill_common import IGNORE
from tests.test_gpu_token_logprobs import entry_points, exact_head

pytestmark = pytest.mark.gpu

LOW = torch.finfo(torch.float32).min


def run(gpu, h, w, b, tok, T, k, ups):
    leaves = [v.to(gpu).requires_grad_(True) for v in (h, w, b)]
    out = entry_points().linear_token_logprobs(leaves[0], leaves[1], tok.to(gpu), leaves[2], 8192, T, k)
    grads = torch.autograd.grad((out.logprobs, out.entropy), leaves, [u.to(gpu) for u in ups])
    return [None if v is None else v.cpu() for v in out], [v.cpu() for v in grads]


def operands(N, V):
    g = torch.Generator().manual_seed(N + V)
    h, w, b = exact_head(g, N, 64, V, True)
    tok = torch.randint(0, V, (N,), generator=g)
    tok[::5] = IGNORE
    tok[1], tok[2] = 3, 4
    return h, w, b, tok, [torch.randn(N, generator=g) for _ in range(2)]


@pytest.mark.parametrize("k", [0, 3])
@pytest.mark.parametrize("T", [0.4, 1.0, 1.3, 3.0])
@pytest.mark.parametrize("N,V", [(6, 300), (300, 1000)])
def test_some_columns(gpu, N, V, T, k):
    """As under a mask of -inf, but for the masked tokens' log-probabilities: LOW / T (less a logsumexp that is far below
    its last place), -inf only where fp32 has no such number."""
    h, w, b, tok, ups = operands(N, V)
    masked = torch.zeros(V, dtype=torch.bool)
    masked[::3] = True
    at = torch.where(tok == IGNORE, False, masked[tok.clamp(min=0)])
    assert at.any() and not at.all()
    got, grads = run(gpu, h, w, b.masked_fill(masked, LOW), tok, T, k, ups)
    want, wgrads = run(gpu, h, w, b.masked_fill(masked, -math.inf), tok, T, k, ups)
    assert torch.equal(got[0][~at], want[0][~at]) and torch.equal(got[1], want[1])
    assert all(torch.equal(p, q) for p, q in zip(grads, wgrads)) and all(v.isfinite().all() for v in grads)
    if k:
        assert torch.equal(got[2], want[2]) and torch.equal(got[3], want[3])
    assert (want[0][at] == -math.inf).all()
    low = LOW / T
    if low < LOW:
        assert (got[0][at] == -math.inf).all()
    else:
        # 1 / T and the product are rounded, and the logits' other terms are below 2^-90 of it
        assert ((got[0][at].double() - low).abs() <= 3 * 2.0 ** -24 * abs(low)).all()


@pytest.mark.parametrize("k", [0, 3])
@pytest.mark.parametrize("T", [0.05, 1.0, 2.0, 1000.0])
@pytest.mark.parametrize("N,V", [(6, 300), (300, 1000), (3, 40000)])
@pytest.mark.parametrize("kind", ["lowest", "low", "one"])
def test_every_column(gpu, N, V, T, k, kind):
    """Rows of which nothing is left: as under a bias of -inf alone, with alternatives and without."""
    h, w, b, tok, ups = operands(N, V)
    b[:] = {"lowest": LOW, "low": -1e34, "one": -math.inf}[kind]
    if kind == "one":
        b[7] = LOW
    got, grads = run(gpu, h, w, b, tok, T, k, ups)
    counts = tok != IGNORE
    assert torch.equal(got[0], torch.where(counts, -math.inf, 0.0)) and not got[1].any()
    assert not any(v.any() for v in grads)
    if k:
        order = [0, 1, 2] if kind != "one" else [7, 0, 1]
        assert torch.equal(got[2], torch.where(counts, -math.inf, 0.0)[:, None].expand(N, k))
        assert torch.equal(got[3], torch.where(counts[:, None], torch.tensor(order), -1))
