"""Layer norm of rows that lie far from 0: what the mean rounds away must not come back as the row's variation."""
import pytest
import torch

from tests.distill_common import DTYPES, half_step

pytestmark = pytest.mark.gpu

EPS = 1e-5


def error(D):
    """Relative error of a sum of D terms by 64 threads or more and a tree, and a few roundings around it."""
    return (D / 64 + 32) * 2.0 ** -24


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("D", [3, 100, 896, 1001, 5000, 9999, 20000])
def test_rows_of_equal_values(gpu, D, dtype):
    """They have no variation: y is the bias, x takes no part in the gradients."""
    from chronicals_amd.kernels.layer_norm import layer_norm
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(D)
    c = torch.tensor([1.1, -3.3, 100.1, 1000.1, -12345.6, 0.1, 65000.0]).to(dt)
    N = len(c)
    x = c[:, None].expand(N, D).contiguous()
    w, b, dy = (torch.randn(s, generator=g).to(dt) for s in ((D,), (D,), (N, D)))
    leaves = [v.to(gpu).requires_grad_(True) for v in (x, w, b)]
    y = layer_norm(*leaves, EPS)
    dx, dw, db = (v.double().cpu() for v in torch.autograd.grad(y, leaves, dy.to(gpu)))
    # the mean is off by error(D) of it, and the mean of the differences from it by
    # error(D) of that, in units of sqrt(eps)
    n = 4 * error(D) ** 2 * c.double().abs()[:, None] / EPS ** 0.5
    rel, least = half_step(dt)
    w, b, dy = w.double(), b.double(), dy.double()
    assert ((y.detach().double().cpu() - b).abs() <= rel * b.abs() + least + n * w.abs() + 2.0 ** -24 * b.abs()).all()
    a = dy * w
    want = (a - a.mean(1, keepdim=True)) / EPS ** 0.5
    mag = (a.abs() + a.abs().mean(1, keepdim=True)) / EPS ** 0.5
    assert ((dx - want).abs() <= rel * want.abs() + least + 4 * error(D) * mag).all()
    assert not dw.any()


@pytest.mark.parametrize("offset", [1e3, -1e4, 1e5])
@pytest.mark.parametrize("D", [100, 896, 1001, 5000, 16384, 20000])
def test_offset_rows(gpu, D, offset):
    """fp32 rows of unit variation around an offset, as far as the row itself holds it."""
    from chronicals_amd.kernels.layer_norm import layer_norm
    g = torch.Generator().manual_seed(D)
    x = torch.randn(9, D, generator=g) + offset
    y = layer_norm(x.to(gpu), None, None, EPS).double().cpu()
    v = x.double()
    m = v.mean(1, keepdim=True)
    n = (v - m) / torch.sqrt(((v - m) ** 2).mean(1, keepdim=True) + EPS)
    # differences from the rounded mean are exact, their mean is off by error(D) of
    # their magnitudes (about 1, and the rounded mean's own shift), and so is their
    # variance
    shift = error(D) * abs(offset)
    assert ((y - n).abs() <= 4 * error(D) * (1 + shift) ** 2 * (1 + n.abs())).all()
