"""RMS norm in 8 bits: q is y / scale, the fp32 quotient, rounded to nearest even, for scales that are no power of two."""
import pytest
import torch

pytestmark = pytest.mark.gpu

MOST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def around_midpoints(dtype, scale, D):
    """Values whose quotients by the scale are the type's midpoints, or lie up to three fp32 steps beside them."""
    codes = torch.arange(0, 0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn).float() if dtype != torch.int8 else \
        torch.arange(0, 128).float()
    mid = ((codes[:-1] + codes[1:]) / 2).double() * float(scale)
    v = mid.float()
    out = [v]
    for way in (float("inf"), -float("inf")):
        u = v
        for _ in range(3):
            u = torch.nextafter(u, torch.tensor(way))
            out.append(u)
    v = torch.cat(out)
    v = torch.cat([v, -v])
    return torch.nn.functional.pad(v, (0, D - v.numel()))


@pytest.mark.parametrize("D", [2048, 20480])  # rows in registers, and longer ones
@pytest.mark.parametrize("xdtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype", list(MOST))
@pytest.mark.parametrize("group", [None, 32, 256])
def test_every_midpoint(gpu, group, dtype, xdtype, D):
    """A row of ones has a mean square of 1, so with eps 0 y is the weight, whose largest value stands in every group."""
    from chronicals_amd.kernels.rms_norm import rms_norm_quantized
    for most in (0.3, 1.0, 3.7, 5.0, 1000.1, 3e-20, 7e19):
        top = torch.tensor(most, dtype=torch.float32)
        scale = top / MOST[dtype]
        w = around_midpoints(dtype, scale, D)
        w = w.clamp(-top, top)
        w[31::32] = top
        q, scales = rms_norm_quantized(torch.ones(1, D, device=gpu, dtype=xdtype), w.to(gpu), None, 0.0, dtype, group)
        assert (scales.cpu() == scale).all(), most
        v = w / scale
        want = torch.round(v) if dtype == torch.int8 else v.clamp(-448, 448).to(dtype).float()
        got = q[0].cpu().float()
        assert torch.equal(got, want), (most, (got != want).nonzero()[:4].tolist())


@pytest.mark.parametrize("dtype", list(MOST))
def test_as_the_rounded_norm(gpu, dtype):
    """fp32 rows: the codes are those of y, which rms_norm gives in fp32, over the scales."""
    from chronicals_amd.kernels.rms_norm import rms_norm, rms_norm_quantized
    g = torch.Generator().manual_seed(3)
    x, w = torch.randn(64, 4096, generator=g), 1 + 0.3 * torch.randn(4096, generator=g)
    y = rms_norm(x.to(gpu), w.to(gpu)).cpu()
    for group in (None, 128):
        q, scales = rms_norm_quantized(x.to(gpu), w.to(gpu), dtype=dtype, group_size=group)
        size = group or 4096
        by = scales.cpu().view(64, -1).repeat_interleave(size, 1)
        assert torch.equal(by[:, ::size], y.abs().view(64, -1, size).amax(2) / MOST[dtype])
        v = y / by
        want = torch.round(v) if dtype == torch.int8 else v.clamp(-448, 448).to(dtype).float()
        assert torch.equal(q.cpu().float(), want)
