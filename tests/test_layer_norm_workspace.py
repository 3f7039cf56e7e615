"""The workspace of layer norm's backward: what the call uses, and no more."""
import ctypes

import pytest
import torch

from chronicals_amd import _lib

P = ctypes.c_void_p(4096)  # an aligned address that nothing reads


def size(fn, *args):
    out = ctypes.c_size_t(0)
    assert fn(*args, ctypes.byref(out)) == 0, _lib.load().cce_last_error()
    return out.value


@pytest.mark.parametrize("dtype", [_lib.CCE_DTYPE_BF16, _lib.CCE_DTYPE_F16, _lib.CCE_DTYPE_F32])
@pytest.mark.parametrize("N,D", [(0, 64), (1, 1), (50, 96), (16384, 896), (1 << 20, 4096), (1 << 20, 16384),
                                 (1024, 20000), (1 << 20, 1 << 20)])
def test_bounds(N, D, dtype):
    lib = _lib.load()
    most = size(lib.cce_layer_norm_backward_workspace_bytes, N, D)
    need = size(lib.cce_layer_norm_backward_workspace_bytes_for, N, D, dtype, 1)
    assert 0 < need <= most
    assert size(lib.cce_layer_norm_backward_workspace_bytes_for, N, D, dtype, 0) == 0
    # dw and db of each workgroup: 768 of a wave per row, 512 of 256 threads a row and 256 of 1024 at most, not more
    # than rows, and 128 MiB
    chunks = -(-D // (4 if dtype == _lib.CCE_DTYPE_F32 else 8))
    parts = 768 if chunks <= 256 else 512 if chunks <= 1024 or D > 16384 else 256
    parts = max(1, min(parts, N, (1 << 24) // D))
    assert need <= 2 * (parts * D * 4 + 256)
    # the entry point asks for as much, and for none without the parameters' gradients
    back = lib.cce_layer_norm_backward
    for dw, db in ((P, None), (None, P), (P, P)):
        assert back(P, P, dtype, D, P, dtype, P, P, N, D, None, dw, db, P, need - 1, None) == _lib.CCE_ERR_WORKSPACE
    assert back(P, P, dtype, D, P, dtype, P, P, N, D, None, None, None, None, 0, None) == _lib.CCE_OK


def test_refusals():
    lib = _lib.load()
    query, out = lib.cce_layer_norm_backward_workspace_bytes_for, ctypes.c_size_t(0)
    for args in ((4, 64, 7, 1), (-1, 64, 0, 1), (4, 0, 0, 1), (4, (1 << 20) + 1, 0, 1)):
        assert query(*args, ctypes.byref(out)) == _lib.CCE_ERR_INVALID_ARG
    assert query(4, 64, 0, 1, None) == _lib.CCE_ERR_INVALID_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,D", [(5000, 896), (600, 4096), (2000, 16384), (300, 20000)])
def test_memory_of_a_backward(gpu, N, D, dtype):
    """A backward allocates its gradients and the parts, and only the gradient where the parameters are frozen; behind
    parts of exactly that size nothing is written."""
    from chronicals_amd.kernels.layer_norm import layer_norm
    lib = _lib.load()
    g = torch.Generator().manual_seed(7)
    x = torch.randn(N, D, generator=g).to(dtype).to(gpu).requires_grad_(True)
    w, b = (torch.randn(D, generator=g).to(dtype).to(gpu) for _ in range(2))
    dy = torch.randn(N, D, generator=g).to(dtype).to(gpu)
    code = _lib.CCE_DTYPE_BF16 if dtype == torch.bfloat16 else _lib.CCE_DTYPE_F32
    need = size(lib.cce_layer_norm_backward_workspace_bytes_for, N, D, code, 1)
    for train in (False, True):
        leaves = [x] + ([w.requires_grad_(True), b.requires_grad_(True)] if train else [])
        y = layer_norm(x, w, b)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        grads = torch.autograd.grad(y, leaves, dy)
        torch.cuda.synchronize()
        extra = torch.cuda.max_memory_allocated() - before
        results = sum(v.numel() * v.element_size() for v in grads)
        # the allocator rounds each block up to 512 bytes, and to 2 MiB where it is large
        assert extra <= results + (need if train else 0) + 4 * (2 << 20), (extra, results, need)
    with torch.no_grad():
        _, mean, rstd = torch.ops.chronicals_hip.layer_norm_fwd(x, w, b, 1e-5)
    dw, db = torch.empty_like(w), torch.empty_like(b)
    ws = torch.full((need + 4096,), 0x5a, dtype=torch.uint8, device=gpu)
    rc = lib.cce_layer_norm_backward(dy.data_ptr(), x.data_ptr(), code, D, w.data_ptr(), code, mean.data_ptr(),
                                     rstd.data_ptr(), N, D, None, dw.data_ptr(), db.data_ptr(), ws.data_ptr(), need,
                                     torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.cce_last_error()
    assert torch.equal(dw, grads[1]) and torch.equal(db, grads[2])
    assert (ws[need:] == 0x5a).all()
