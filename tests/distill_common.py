"""References in 64 bits and inputs of the distillation, top-logits and layer-norm tests."""
import math

import torch

IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# Relative error of an exponential or a quotient of them in fp32.  The exponent
# (x - m) log2(e) / T - log2(s) is below 150 in magnitude where its power does not
# vanish; three operations round it, each by at most 2^-24 of it, and a few more
# round the result: (8 + 4 * 150) 2^-24 < 2^-14.
EXP_ERR = 2.0 ** -14
# The hardware's exponential gives 0 where the result would be subnormal: up to
# 2^-126 is lost of each, before it is scaled by the weights.
EXP_LEAST = 2.0 ** -126


def half_step(dtype):
    """Largest relative error of one rounding, and the absolute one where the type goes subnormal."""
    return torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def teacher(g, N, V, K, pad=0.0, dtype=torch.float32, index_dtype=torch.int64):
    """Entries with distinct columns in each row; `pad`: share of entries that are padding, which hold NaN."""
    index = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(N)]) if N else torch.zeros(0, K).long()
    t = torch.randn(N, K, generator=g) * 3
    out = torch.rand(N, K, generator=g) < pad
    return t.masked_fill(out, math.nan).to(dtype), index.masked_fill(out, -1).to(index_dtype)


def labels(g, N, V, ignored=0.2):
    lab = torch.randint(0, V, (N,), generator=g)
    lab[torch.rand(N, generator=g) < ignored] = IGNORE
    return lab


def reference(x, t, index, lab=None, T=1.0, kd=1.0, ce=0.0):
    """(row losses, gradient of each row's loss, which rows count, magnitudes of the losses' and gradients' terms) for
    student logits x, in 64 bits, row by row."""
    x, t = x.double(), t.double()
    N, V = x.shape
    rows, grad = torch.zeros(N, dtype=torch.float64), torch.zeros(N, V, dtype=torch.float64)
    mag_rows, mag = rows.clone(), grad.clone()
    counts = torch.zeros(N, dtype=torch.bool)
    for n in range(N):
        entries = [(int(c), float(v)) for c, v in zip(index[n], t[n]) if 0 <= int(c) < V and not float(v) == -math.inf]
        counts[n] = bool(entries) if lab is None else int(lab[n]) != IGNORE
        if not counts[n]:
            continue
        if entries and kd:
            v = torch.tensor([e[1] for e in entries], dtype=torch.float64)
            log_q = torch.log_softmax((v - v.max()) / T, 0)
            log_p = torch.log_softmax(x[n] / T, 0)
            grad[n] += kd * T * log_p.exp()
            mag[n] += kd * T * log_p.exp()
            for (c, _), lq in zip(entries, log_q):
                q = math.exp(lq)
                if q == 0.0:
                    continue
                rows[n] += kd * T * T * q * (lq - log_p[c])
                mag_rows[n] += abs(kd) * T * T * q * (abs(lq) + abs(log_p[c]) + 1)
                grad[n, c] -= kd * T * q
                mag[n, c] += abs(kd) * T * q
        if ce:
            log_p = torch.log_softmax(x[n], 0)
            grad[n] += ce * log_p.exp()
            mag[n] += abs(ce) * log_p.exp()
            rows[n] += ce * torch.logsumexp(x[n], 0)
            mag_rows[n] += abs(ce) * (torch.logsumexp(x[n], 0).abs() + 1)
            c = int(lab[n])
            if 0 <= c < V:
                rows[n] -= ce * x[n, c]
                mag_rows[n] += abs(ce) * abs(x[n, c])
                grad[n, c] -= ce
                mag[n, c] += abs(ce)
    return rows, grad, counts, mag_rows, mag


def close(got, want, tol, what=""):
    """Elementwise |got - want| <= tol, with infinities and NaN alike."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~same & ~((got - want).abs() <= tol)
    if bad.any():
        at = tuple(i[0].item() for i in bad.nonzero(as_tuple=True))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {at}: {got[at]} for {want[at]}, "
                             f"tolerance {torch.as_tensor(tol).expand(want.shape)[at]}")
