"""Log-probabilities from hidden states of more than 16384 rows: the unit that the logits' gradient is held in is found by
a launch of its own, over all rows."""
import pytest
import torch

from tests.logprobs_common import tokens
from tests.test_gpu_token_logprobs import check_linear, entry_points, head

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,V,T,bias,frozen", [(16384, 300, 1.0, False, False), (16385, 300, 1.0, False, False),
                                               (16385, 257, 0.8, True, False), (20000, 100, 1.0, False, True)])
def test_against_64_bits(gpu, N, V, T, bias, frozen):
    g = torch.Generator().manual_seed(N + V)
    h, w = head(g, N, 64, V)
    b = torch.randn(V, generator=g) if bias else None
    check_linear(gpu, h, w, tokens(g, N, V, 0.3), b, T, 0, frozen)


@pytest.mark.parametrize("N", [16384, 16385, 17409])
@pytest.mark.parametrize("row", ["first", "last"])
def test_one_row_has_the_largest_gradient(gpu, N, row):
    """All gradients are 0 but one row's, 1.7.  In the unit of that one, its share at the token, 1.7 (1 - p) with p below
    2^-10, is held as 1.7: off by p.  In a unit found without that row it would be rounded to 1.6953 or 1.7031, off by
    2^-9."""
    g = torch.Generator().manual_seed(2)
    V, d, n = 2048, 64, 0 if row == "first" else N - 1
    h, w = torch.randn(N, d, generator=g).bfloat16(), (torch.randn(V, d, generator=g) * 0.01).bfloat16()
    tok = torch.randint(0, V, (N,), generator=g)
    p = torch.softmax(h[n].double() @ w.double().t(), 0)[tok[n]].item()
    assert p < 2.0 ** -10
    up = torch.zeros(N)
    up[n] = 1.7
    wg = w.float().to(gpu).requires_grad_(True)
    out = entry_points().linear_token_logprobs(h.to(gpu), wg, tok.to(gpu))
    (dw,) = torch.autograd.grad(out.logprobs, wg, up.to(gpu))
    want = up[n].double() * (1 - p) * h[n].double()
    # p itself, and a few roundings of fp32
    assert ((dw[tok[n]].double().cpu() - want).abs() <= (p + 2.0 ** -20) * 1.7 * h[n].double().abs()).all()
