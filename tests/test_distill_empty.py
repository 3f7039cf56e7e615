"""An empty batch with labels: the labels are given, though their tensor has no storage."""
import ctypes

import pytest
import torch

from chronicals_amd import _lib

P = ctypes.c_void_p(4096)  # an aligned address that nothing reads


def test_c_entry_points_take_no_rows_with_labels():
    """N = 0, null labels and a weight of their loss: the call goes on to the check behind this one.  With rows it is
    refused."""
    lib = _lib.load()
    teacher = ctypes.byref(_lib.Teacher(logits=None, indices=None, entries=4, logits_dtype=1, indices_int64=1,
                                        temperature=1.0, distill_weight=0.5, ce_weight=0.5))
    small = _lib.CCE_ERR_WORKSPACE
    assert lib.cce_distill_logits_forward(None, 1, 100, teacher, None, 0, 0, 100, -100, 1, P, None, P, P, 8,
                                          None) == small, lib.cce_last_error()
    assert lib.cce_distill_forward(None, None, None, teacher, None, 0, 0, 64, 100, -100, 1, P, None, None, None, P, P, 8,
                                   None) == small, lib.cce_last_error()
    assert lib.cce_distill_logits_backward(None, None, 1, 100, teacher, None, 0, None, None, 0, 100, -100, 1, None, 100,
                                           None) == _lib.CCE_OK, lib.cce_last_error()
    assert lib.cce_distill_backward(None, None, None, None, teacher, None, None, None, None, 0, 64, 100, 1, 0, None, 0,
                                    None, 0, None, P, 1 << 30, None) == _lib.CCE_OK, lib.cce_last_error()
    full = ctypes.byref(_lib.Teacher(logits=4096, indices=4096, entries=4, logits_dtype=1, indices_int64=1,
                                     temperature=1.0, distill_weight=0.5, ce_weight=0.5))
    assert lib.cce_distill_logits_forward(P, 1, 100, full, None, 0, 1, 100, -100, 1, P, P, P, P, 1 << 30,
                                          None) == _lib.CCE_ERR_INVALID_ARG
    assert b"needs labels" in lib.cce_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("index_dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_empty_batch_with_labels(gpu, reduction, index_dtype):
    from chronicals_amd.kernels import distillation as D
    t, index = torch.zeros(0, 4, device=gpu), torch.zeros(0, 4, device=gpu, dtype=index_dtype)
    lab = torch.zeros(0, device=gpu, dtype=index_dtype)
    x = torch.zeros(0, 100, device=gpu, requires_grad=True)
    h = torch.zeros(0, 64, device=gpu, dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(100, 64, device=gpu, dtype=torch.bfloat16, requires_grad=True)
    b = torch.ones(100, device=gpu, requires_grad=True)
    how = dict(temperature=2.0, distill_weight=0.5, ce_weight=0.5, reduction=reduction)
    losses = [D.distillation_loss(x, t, index, lab, **how),
              D.linear_distillation_loss(h, w, t, index, lab, b, **how)]
    for loss in losses:
        assert loss.shape == ((0,) if reduction == "none" else ())
        assert reduction == "none" or loss.item() == 0.0
    dx, dh, dw, db = torch.autograd.grad([v.sum() for v in losses], [x, h, w, b])
    assert dx.shape == x.shape and dh.shape == h.shape and not dw.any() and not db.any()
