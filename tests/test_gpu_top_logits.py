"""The k largest logits of each row, exactly."""
import math

import pytest
import torch

from tests.distill_common import DTYPES

pytestmark = pytest.mark.gpu


def want(x, k):
    """Stable descending order: equal values by the lower index first, NaN first, -0 equal to +0."""
    v = (x.double() + 0.0).masked_fill(x.isnan(), math.inf)
    order = torch.argsort(v + 0.0, dim=-1, descending=True, stable=True)
    # NaN before +inf
    nan = torch.gather(x.isnan(), -1, order)
    order = torch.gather(order, -1, torch.argsort(nan.int(), dim=-1, descending=True, stable=True))[..., :k]
    return torch.gather(x, -1, order), order


def check(gpu, x, k, on=None):
    from chronicals_amd.kernels.distillation import top_logits
    values, indices = top_logits(x.to(gpu) if on is None else on, k)
    wv, wi = want(x, k)
    assert values.dtype == x.dtype and indices.dtype == torch.int64 and values.shape == wv.shape
    assert torch.equal(indices.cpu(), wi)
    bits = {2: torch.int16, 4: torch.int32}[x.element_size()]
    assert torch.equal(values.cpu().view(bits), wv.view(bits))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("N,V,k", [(1, 1, 1), (3, 5, 5), (2, 255, 1), (4, 256, 256), (5, 257, 256), (3, 1000, 17),
                                   (7, 4099, 64), (2, 50257, 100), (1, 151936, 256), (300, 2111, 33), (1100, 700, 9)])
def test_random(gpu, N, V, k, dtype):
    g = torch.Generator().manual_seed(N + V + k)
    check(gpu, (torch.randn(N, V, generator=g) * 2).to(DTYPES[dtype]), k)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_rows_of_equal_values(gpu, dtype):
    dt = DTYPES[dtype]
    V = 30011
    g = torch.Generator().manual_seed(0)
    x = torch.zeros(10, V)
    x[1] = -math.inf
    x[2, 20000:] = 1.0                              # ties that begin late
    x[3] = torch.randint(0, 3, (V,), generator=g).float()
    x[4] = torch.arange(V) % 2 * -0.0               # zeros of both signs
    x[5, ::7] = math.nan
    x[5, 3] = math.inf
    x[6] = torch.finfo(dt).min
    x[6, 29999] = torch.finfo(dt).max
    x[7, 4000:4200] = 5.0
    x[7, 100] = 6.0
    x[8] = torch.arange(V).float().flip(0) / 64
    x[9] = torch.arange(V).float() / 64
    for k in (1, 64, 200, 256):
        check(gpu, x.to(dt), k)


def test_largest_in_one_place(gpu):
    """Every large value within one run of columns, or at one stride."""
    V = 100000
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, V, generator=g)
    x[0, 5000:5300] += 20
    x[1, ::256] += 20
    x[2, 7::1024] += 20
    x[3, ::2048] += 20
    x[4, ::4096] += 20
    x[5, -300:] += 20
    for dt in (torch.bfloat16, torch.float32):
        for k in (64, 256):
            check(gpu, x.to(dt), k)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_masked_rows(gpu, dtype):
    """Fewer values than k beside a mask's value, which fills the rest by the lowest columns; the mask's value may be
    -inf, the type's lowest, zero of either sign or any other, and stand late in the row."""
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(4)
    V = 60013
    for mask in (-math.inf, torch.finfo(dt).min, 0.0, -0.0, 1.25, -7.3, math.inf, math.nan):
        x = torch.full((6, V), mask)
        for n, kept in enumerate((1, 5, 40, 63, 300)):
            at = torch.randperm(V, generator=g)[:kept]
            x[n, at] = torch.randn(kept, generator=g) + (20 if n % 2 else 0)
        x[5, :50000] = -2e4
        for k in (1, 64, 256):
            check(gpu, x.to(dt), k)


def test_strided_rows_and_shapes(gpu):
    g = torch.Generator().manual_seed(2)
    big = torch.randn(6, 5007, generator=g).bfloat16()
    check(gpu, big[:, 3:5004], 40, big.to(gpu)[:, 3:5004])
    check(gpu, big[:, 3:5004], 40, big[:, 3:5004].t().contiguous().to(gpu).t())
    check(gpu, big[:1].expand(6, -1).contiguous(), 40, big[:1].to(gpu).expand(6, -1))
    check(gpu, big.view(2, 3, -1), 7)
    check(gpu, big[0], 7)


def test_no_rows(gpu):
    from chronicals_amd.kernels.distillation import top_logits
    values, indices = top_logits(torch.zeros(0, 50, device=gpu), 5)
    assert values.shape == indices.shape == (0, 5)


def test_captured_and_replayed(gpu):
    from chronicals_amd.kernels.distillation import top_logits
    g = torch.Generator().manual_seed(3)
    a, b = (torch.randn(3, 40000, generator=g).to(gpu) for _ in range(2))
    x = a.clone()
    top_logits(x, 50)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = top_logits(x, 50)
    for turn in range(4):
        x.copy_(b if turn % 2 else a)
        graph.replay()
        got = [v.clone() for v in out]
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, top_logits(x, 50)))
