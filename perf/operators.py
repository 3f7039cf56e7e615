"""Performance cases of the distillation and normalisation operators.

A case is one call that a training or evaluation program makes.  ``run`` computes
it in plain torch operations in 32 bits, or, where ``own`` is set, by the
framework's entry points on the same inputs; ``exact`` gives the outputs in 64
bits from the definitions.  Kinds:

  kd         distillation from a teacher's top logits (and cross-entropy with the
             labels, where ce is not 0) over student logits that exist: loss and
             gradient of the logits
  kd_eval    the same loss per row, without a gradient
  kd_linear  the same loss from hidden states and the head's weight: loss and
             gradients of hidden, weight (unless frozen) and bias
  top        a teacher's k largest logits of each row and where they are
  ln         layer norm over the last dimension, forward and backward
  ln_eval    its forward alone

Per row, over the teacher's usable entries (logit t_k at index i_k, padding has
index -1), with temperature T:
  q = softmax(t / T);  loss = kd T^2 sum_k q_k (log q_k - log softmax(x / T)[i_k])
                              + ce (logsumexp(x) - x[label])
averaged over the rows that count: those with a label other than -100, or, where
the call has no labels, those with a usable entry.
"""
import math

import torch

own = False

IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _kd(kind, N, V, K, dtype="bf16", T=1.0, kd=1.0, ce=0.0, labels=False, ignored=0.0, pad=0.0, d=0, frozen=False,
        bias=False):
    """ignored: share of labels that are -100; pad: share of the rows whose teacher gives fewer than K entries (one in
    four of these gives none)."""
    return {"kind": kind, "N": N, "V": V, "K": K, "dtype": dtype, "T": T, "kd": kd, "ce": ce, "labels": labels,
            "ignored": ignored, "pad": pad, "d": d, "frozen": frozen, "bias": bias}


def _top(N, V, K, dtype="bf16"):
    return {"kind": "top", "N": N, "V": V, "K": K, "dtype": dtype}


def _ln(kind, N, D, dtype="bf16", wdtype="bf16", bias=True):
    return {"kind": kind, "N": N, "D": D, "dtype": dtype, "wdtype": wdtype, "bias": bias}


def listed():
    return [
        # a model that returns logits, distilled with the labels' loss beside: two sequences of 2048 tokens
        dict(_kd("kd", 4096, 151936, 64, T=2.0, kd=0.5, ce=0.5, labels=True, ignored=0.05), name="kd_4096"),
        # GPT-2-sized vocabulary, rows that start off alignment, a top-p teacher with ragged entries, no labels
        dict(_kd("kd", 2047, 50257, 100, T=4.0, pad=0.3), name="kd_ragged"),
        # a short continuation's rows in fp32: launches count
        dict(_kd("kd", 16, 151936, 32, "fp32"), name="kd_16_fp32"),
        # held-out divergence from the teacher, prompt tokens (40%) masked
        dict(_kd("kd_eval", 1024, 128256, 64, T=1.0, labels=True, ignored=0.4), name="kd_eval"),
        # fused with the head: one short chat turn on a small vocabulary
        dict(_kd("kd_linear", 64, 32000, 16, T=2.0, labels=True, ignored=0.05, d=896), name="kd_linear_64"),
        # one 2048-token sequence, both losses
        dict(_kd("kd_linear", 2048, 151936, 64, T=2.0, kd=0.5, ce=0.5, labels=True, ignored=0.05, d=896),
             name="kd_linear_2048"),
        # wide hidden, 128k vocabulary: the largest
        dict(_kd("kd_linear", 8192, 128256, 64, T=1.0, kd=0.7, ce=0.3, labels=True, ignored=0.02, d=4096),
             name="kd_linear_8192"),
        # hidden size that is no multiple of 64, bias, a ragged teacher, no labels
        dict(_kd("kd_linear", 1500, 50257, 50, T=3.0, pad=0.3, d=1000, bias=True), name="kd_linear_ragged"),
        # a teacher's logits of one 2048-token sequence, kept as the 64 largest
        dict(_top(2048, 151936, 64), name="top_2048"),
        # a few rows in fp32
        dict(_top(16, 128256, 128, "fp32"), name="top_16_fp32"),
        # the norm before the head of the 0.5B-parameter benchmark model, 16384 tokens
        dict(_ln("ln", 16384, 896), name="ln_16384"),
        # a short turn in evaluation
        dict(_ln("ln_eval", 64, 768, "fp32", "fp32"), name="ln_eval_64"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["kd", "kd", "kd_eval", "kd_linear", "kd_linear", "kd_linear", "top", "top", "ln", "ln", "ln_eval"])
    if kind in ("ln", "ln_eval"):
        D = _log(rng, 1, 256) * 64 if rng.random() < 0.6 else _log(rng, 16, 20000)
        N = _log(rng, 1, min(65536, 65536 * 4096 // D))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return _ln(kind, N, D, dtype, rng.choice([dtype, "fp32"]), rng.random() < 0.8)
    V = _log(rng, 1000, 152064)
    K = _log(rng, 1, 256)
    if kind == "top":
        return _top(_log(rng, 1, min(8192, 2048 * 151936 // V)), V, K, rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    T = rng.choice([1.0, 1.0, 1.5, 2.0, 4.0])
    kd, ce, labels = rng.choice([(1.0, 0.0, False), (1.0, 0.0, True), (0.5, 0.5, True), (0.9, 0.1, True)])
    more = dict(T=T, kd=kd, ce=ce, labels=labels, ignored=rng.choice([0.0, 0.05, 0.4]) if labels else 0.0,
                pad=rng.choice([0.0, 0.0, 0.3]))
    if kind == "kd_linear":
        # hidden sizes of models are mostly multiples of 64; the head's product is computed in bf16
        d = _log(rng, 2, 64) * 64 if rng.random() < 0.7 else _log(rng, 16, 256) * 8 + 8
        N = _log(rng, 1, min(16384, 8192 * 4096 * 128256 // (2 * d * V)))
        return _kd(kind, N, V, K, d=d, frozen=rng.random() < 0.3, bias=rng.random() < 0.2, **more)
    N = _log(rng, 1, min(16384, 4096 * 151936 // (2 * V)))
    return _kd(kind, N, V, K, rng.choice(["bf16", "bf16", "fp16", "fp32"]), **more)


def _teacher(case, g, dev):
    """Distinct indices per row and descending logits, with padding behind the entries of a ragged row."""
    N, V, K = case["N"], case["V"], case["K"]
    first = torch.randint(0, V, (N, 1), generator=g, device=dev)
    step = torch.randint(1, V // K + 1, (N, 1), generator=g, device=dev)
    index = (first + step * torch.arange(K, device=dev)) % V
    t = torch.randn(N, K, generator=g, device=dev).sort(1, descending=True).values * 3 + 10
    if case["pad"]:
        short = torch.rand(N, 1, generator=g, device=dev) < case["pad"]
        none = torch.rand(N, 1, generator=g, device=dev) < 0.25
        keep = torch.randint(1, K + 1, (N, 1), generator=g, device=dev).masked_fill(none, 0)
        index = torch.where(short & (torch.arange(K, device=dev) >= keep), -1, index)
    return t.to(DTYPES[case["dtype"]]), index


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s, dt, N = {"case": case}, DTYPES[case["dtype"]], case["N"]
    if case["kind"] in ("ln", "ln_eval"):
        # hidden states: features of unlike scales around a common offset; weights near 1
        D, wdt = case["D"], DTYPES[case["wdtype"]]
        s["x"] = (randn(N, D) * torch.exp(0.5 * randn(D)) + 0.3).to(dt)
        s["w"] = (1 + 0.2 * randn(D)).to(wdt)
        s["b"] = (0.2 * randn(D)).to(wdt) if case["bias"] else None
        if case["kind"] == "ln":
            s["dy"] = randn(N, D).to(dt)
            for name in ("x", "w", "b"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
        return s
    V = case["V"]
    if case["kind"] == "top":
        s["x"] = (randn(N, V) * 2).to(dt)
        return s
    if case["kind"] == "kd_linear":
        # after a final norm, and a usual initialisation of the head
        s["h"] = randn(N, case["d"]).to(dt).requires_grad_(True)
        s["w"] = (randn(V, case["d"]) * 0.02).to(dt).requires_grad_(not case["frozen"])
        s["b"] = (randn(V) * 0.1).to(dt).requires_grad_(not case["frozen"]) if case["bias"] else None
    else:
        s["x"] = (randn(N, V) * 2).to(dt).requires_grad_(case["kind"] == "kd")
    s["t"], s["i"] = _teacher(case, g, dev)
    s["labels"] = None
    if case["labels"]:
        s["labels"] = torch.randint(0, V, (N,), generator=g, device=dev)
        s["labels"][torch.rand(N, generator=g, device=dev) < case["ignored"]] = IGNORE
    return s


def _kd_rows(case, x, t, index, labels):
    """Row losses, the gradient of each with respect to its logits x (32 bits), and which rows count."""
    T, kd, ce = case["T"], case["kd"], case["ce"]
    usable = index >= 0
    at = index.clamp(min=0)
    some = usable.any(1, keepdim=True)
    counts = some[:, 0] if labels is None else labels != IGNORE
    t = torch.where(usable, t.float() / T, -math.inf)
    t = t - torch.where(some, t.amax(1, keepdim=True), 0.0)
    e = torch.exp(t)
    z = e.sum(1, keepdim=True)
    q = torch.where(some, e / z, 0.0)
    log_q = torch.where(usable, t - torch.log(z), 0.0)
    top = x.amax(1, keepdim=True)
    e = torch.exp((x - top) / T)
    z = e.sum(1, keepdim=True)
    xk = (x.gather(1, at) - top) / T
    loss = kd * T * T * (q * (log_q - xk + torch.log(z))).sum(1)
    grad = e * (kd * T / z) * some
    if ce:
        if T != 1.0:
            e = torch.exp(x - top)
            z = e.sum(1, keepdim=True)
        lab = torch.where(counts, labels, 0)[:, None]
        loss = loss + ce * (torch.log(z) + top - x.gather(1, lab))[:, 0]
        grad = grad + e * (ce / z)
        grad.scatter_add_(1, lab, torch.full_like(z, -ce))
    grad.scatter_add_(1, at, q * (-kd * T))
    return torch.where(counts, loss, 0.0), grad * counts[:, None], counts


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind in ("ln", "ln_eval"):
        x, w = s["x"].float(), s["w"].float()
        c = x - x.mean(1, keepdim=True)
        r = torch.rsqrt((c * c).mean(1, keepdim=True) + 1e-5)
        n = c * r
        y = n * w
        if s["b"] is not None:
            y = y + s["b"].float()
        y = y.to(s["x"].dtype)
        if kind == "ln_eval":
            return {"y": y}
        dy = s["dy"].float()
        dn = dy * w
        dx = r * (dn - dn.mean(1, keepdim=True) - n * (dn * n).mean(1, keepdim=True))
        out = {"y": y, "dx": dx.to(s["x"].dtype), "dw": (dy * n).sum(0).to(s["w"].dtype)}
        if s["b"] is not None:
            out["db"] = dy.sum(0).to(s["b"].dtype)
        return out
    if kind == "top":
        v, i = torch.sort(s["x"], dim=1, descending=True, stable=True)
        return {"values": v[:, :case["K"]].contiguous(), "indices": i[:, :case["K"]].contiguous()}
    if kind != "kd_linear":
        loss, grad, counts = _kd_rows(case, s["x"].float(), s["t"], s["i"], s["labels"])
        if kind == "kd_eval":
            return {"loss": loss}
        n = counts.sum().clamp(min=1)
        return {"loss": loss.sum() / n, "dx": (grad / n).to(s["x"].dtype)}
    h, w = s["h"].float(), s["w"].float()
    x = h @ w.t()
    if s["b"] is not None:
        x = x + s["b"].float()
    loss, grad, counts = _kd_rows(case, x, s["t"], s["i"], s["labels"])
    n = counts.sum().clamp(min=1)
    grad = grad / n
    out = {"loss": loss.sum() / n, "dh": (grad @ w).to(s["h"].dtype)}
    if not case["frozen"]:
        out["dw"] = (grad.t() @ h).to(s["w"].dtype)
        if s["b"] is not None:
            out["db"] = grad.sum(0).to(s["b"].dtype)
    return out


def _own(s):
    from chronicals_amd.kernels.distillation import distillation_loss, linear_distillation_loss, top_logits
    from chronicals_amd.kernels.layer_norm import layer_norm

    case = s["case"]
    kind = case["kind"]
    if kind == "ln_eval":
        with torch.no_grad():
            return {"y": layer_norm(s["x"], s["w"], s["b"])}
    if kind == "ln":
        y = layer_norm(s["x"], s["w"], s["b"])
        leaves = {"dx": s["x"], "dw": s["w"], "db": s["b"]}
        leaves = {k: v for k, v in leaves.items() if v is not None}
        return {"y": y.detach(), **dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), s["dy"])))}
    if kind == "top":
        values, indices = top_logits(s["x"], case["K"])
        return {"values": values, "indices": indices}
    how = dict(labels=s["labels"], temperature=case["T"], distill_weight=case["kd"], ce_weight=case["ce"])
    if kind == "kd_eval":
        with torch.no_grad():
            return {"loss": distillation_loss(s["x"], s["t"], s["i"], reduction="none", **how)}
    if kind == "kd":
        loss = distillation_loss(s["x"], s["t"], s["i"], **how)
        return {"loss": loss.detach(), "dx": torch.autograd.grad(loss, s["x"])[0]}
    loss = linear_distillation_loss(s["h"], s["w"], s["t"], s["i"], bias=s["b"], **how)
    leaves = {"dh": s["h"]}
    if not case["frozen"]:
        leaves["dw"] = s["w"]
        if s["b"] is not None:
            leaves["db"] = s["b"]
    return {"loss": loss.detach(), **dict(zip(leaves, torch.autograd.grad(loss, list(leaves.values()))))}


def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return _plain(s)


def work(case):
    """Each input read once and each output written once; the products over the rows that count."""
    kind, N, size = case["kind"], case["N"], SIZE[case["dtype"]]
    if kind in ("ln", "ln_eval"):
        D = case["D"]
        params = (2 if case["bias"] else 1) * D * SIZE[case["wdtype"]]
        if kind == "ln_eval":
            return {"bytes": 2 * N * D * size + params, "flops": 8 * N * D}
        return {"bytes": 4 * N * D * size + 2 * params, "flops": 20 * N * D}
    V, K = case["V"], case["K"]
    if kind == "top":
        return {"bytes": N * V * size + N * K * (size + 8), "flops": N * V}
    entries = N * K * (size + 8) + (8 * N if case["labels"] else 0)
    live = N * (1.0 - (case["ignored"] if case["labels"] else 0.25 * case["pad"]))
    if kind == "kd_linear":
        d = case["d"]
        read, written = (live * d + V * d) * size, N * d * size
        products = 2
        if not case["frozen"]:
            products, written = 3, written + V * d * size + (V * size if case["bias"] else 0)
        return {"bytes": int(read + written + entries), "flops": int(2 * products * live * d * V + 4 * live * K * d)}
    if kind == "kd_eval":
        return {"bytes": int(live * V * size + entries + 4 * N), "flops": int(4 * live * V)}
    return {"bytes": int((live + N) * V * size + entries), "flops": int(8 * live * V)}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("ln", "ln_eval"):
        x, w = s["x"].detach().double(), s["w"].detach().double()
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        n = (x - mean) / torch.sqrt(var + 1e-5)
        y = n * w + (0.0 if s["b"] is None else s["b"].detach().double())
        if kind == "ln_eval":
            return {"y": y}
        dy = s["dy"].double()
        # the projection of dy * w off the constant and the normalised row
        a = dy * w
        dx = (a - (a.sum(1, keepdim=True) + n * (a * n).sum(1, keepdim=True)) / x.shape[1]) / torch.sqrt(var + 1e-5)
        out = {"y": y, "dx": dx, "dw": torch.einsum("nd,nd->d", dy, n)}
        if s["b"] is not None:
            out["db"] = dy.sum(0)
        return out
    if kind == "top":
        # one integer per element that orders by value and, among equals, by the lower index first
        x = s["x"].float() + 0.0
        bits = x.view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) - torch.arange(case["V"], device=x.device)
        at = key.topk(case["K"], 1).indices
        return {"values": s["x"].double().gather(1, at), "indices": at}
    N, V, T, kd, ce = case["N"], case["V"], case["T"], case["kd"], case["ce"]
    linear, with_grad = kind == "kd_linear", kind != "kd_eval"
    usable = s["i"] >= 0
    at = torch.where(usable, s["i"], 0)
    labels = s["labels"]
    counts = usable.any(1) if labels is None else labels != IGNORE
    n = max(int(counts.sum()), 1)
    log_q = torch.log_softmax((s["t"].double() / T).masked_fill(~usable, -1e300), 1)
    q = torch.exp(log_q) * usable
    if linear:
        h, w = s["h"].detach().double(), s["w"].detach().double()
        dh, dw = torch.zeros_like(h), torch.zeros_like(w)
        db = torch.zeros(V, dtype=torch.float64, device=h.device)
    rows = torch.zeros(N, dtype=torch.float64, device=at.device)
    dx = torch.empty(N, V, dtype=torch.float64, device=at.device) if kind == "kd" else None
    for a in range(0, N, 2048):
        r = slice(a, min(a + 2048, N))
        if linear:
            x = h[r] @ w.t()
            if s["b"] is not None:
                x += s["b"].detach().double()
        else:
            x = s["x"][r].detach().double()
        c = counts[r].double()[:, None]
        lp = torch.log_softmax(x / T, 1)
        rows[r] = kd * T * T * (q[r] * (log_q[r].masked_fill(~usable[r], 0.0) - lp.gather(1, at[r]))).sum(1)
        if with_grad:
            grad = lp.exp_().mul_(kd * T * q[r].sum(1, keepdim=True))
            grad.scatter_add_(1, at[r], -kd * T * q[r])
        if ce:
            lp = torch.log_softmax(x, 1)
            lab = labels[r].clamp(min=0)[:, None]
            rows[r] -= ce * lp.gather(1, lab)[:, 0]
            if with_grad:
                grad.add_(lp.exp_(), alpha=ce)
                grad.scatter_add_(1, lab, torch.full_like(c, -ce))
        if not with_grad:
            continue
        grad *= c / n
        if not linear:
            dx[r] = grad
            continue
        dh[r] = grad @ w
        if not case["frozen"]:
            dw.addmm_(grad.t(), h[r])
            db += grad.sum(0)
    rows *= counts
    if kind == "kd_eval":
        return {"loss": rows}
    out = {"loss": rows.sum() / n}
    if not linear:
        out["dx"] = dx
        return out
    out["dh"] = dh
    if not case["frozen"]:
        out["dw"] = dw
        if s["b"] is not None:
            out["db"] = db
    return out
