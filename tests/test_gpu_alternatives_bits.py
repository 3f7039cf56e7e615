"""The alternatives' log-probabilities of few rows, which are split over workgroups and joined: the same bits on every run,
and equal ones for equal logits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SIZES = [(8, 128256, 20), (1, 151936, 20), (3, 50000, 40), (16, 32003, 5)]


def entry_points():
    from chronicals_amd.kernels import token_logprobs
    return token_logprobs


def logits(gpu, N, V, dtype):
    g = torch.Generator().manual_seed(N + V)
    return (torch.randn(N, V, generator=g) * 3).to(dtype).to(gpu), torch.randint(0, V, (N,), generator=g).to(gpu)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,V,k", SIZES)
def test_same_bits_on_every_run(gpu, N, V, k, dtype):
    x, tok = logits(gpu, N, V, dtype)
    f = entry_points().token_logprobs
    first = f(x, tok, 0.8, k)
    for _ in range(40):
        again = f(x, tok, 0.8, k)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,V,k", SIZES)
def test_equal_logits_have_equal_log_probabilities(gpu, N, V, k, dtype):
    x, tok = logits(gpu, N, V, dtype)
    at = torch.arange(k, device=gpu) * (V // k) + 7
    x[:, at] = 20.0
    for T in (0.7, 0.8, 1.0, 1.3, 2.0):
        out = entry_points().token_logprobs(x, tok, T, k)
        assert torch.equal(out.top_indices, at.expand(N, k))
        assert torch.equal(out.top_logprobs, out.top_logprobs[:, :1].expand(N, k)), T


@pytest.mark.parametrize("N", [1, 8])
def test_from_hidden_states(gpu, N):
    g = torch.Generator().manual_seed(N)
    h, w = torch.randn(N, 64, generator=g).bfloat16().to(gpu), (torch.randn(60000, 64, generator=g) * 0.3).bfloat16().to(gpu)
    tok = torch.randint(0, 60000, (N,), generator=g).to(gpu)
    f = entry_points().linear_token_logprobs
    first = f(h, w, tok, top_k=20)
    for _ in range(40):
        assert all(torch.equal(a, b) for a, b in zip(first, f(h, w, tok, top_k=20)))
