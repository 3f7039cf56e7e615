"""Performance cases of the token log-probabilities and of the RMS norm.

A case is one call that a training, scoring or serving program makes.  ``run``
computes it in plain torch operations in 32 bits, or, where ``own`` is set, by the
framework's entry points on the same inputs; ``exact`` gives the outputs in 64 bits
from the definitions.  Kinds:

  lp          log-probabilities of given tokens and entropies over logits that
              exist: both, and the gradient of the logits for given gradients of both
  lp_top      the same without a gradient, and the K largest logits of each row: where
              they are and their log-probabilities
  lp_linear   as lp, from hidden states and the head's weight: gradients of hidden,
              weight (unless frozen) and bias
  lp_linear_top   as lp_top, from hidden states and the head's weight
  rms         RMS norm with the residual's addition, forward and backward
  rms_eval    its forward alone
  rms_q       its forward with an 8-bit output (e4m3 or int8) and scales per row or
              per group of columns

Per row, with z = x / T:  lse = logsumexp(z),  p = exp(z - lse),
  logprob = z[token] - lse,  entropy = -sum p log p,
  dx_v = (g ([v = token] - p_v) - h p_v (log p_v + entropy)) / T
for the gradients g and h of the two; a token of -100 gives 0 and a zero gradient.

RMS norm: s = x + residual, rounded to the residual's type, n = s / sqrt(mean(s^2) + eps),
y = n w.  In 8 bits: scale = max(amax(|y|), 1e-30) / M with M = 448 (e4m3) or 127 (int8) and
q = round(y / scale).
"""
import math

import torch

own = False

IGNORE = -100
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn,
          "int8": torch.int8}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1, "int8": 1}
LARGEST = {"e4m3": 448.0, "int8": 127.0}


def _lp(kind, N, V, dtype="bf16", T=1.0, K=0, ignored=0.0, d=0, frozen=False, bias=False):
    """ignored: share of the tokens that are -100 (a prompt's, padding)."""
    return {"kind": kind, "N": N, "V": V, "dtype": dtype, "T": T, "K": K, "ignored": ignored, "d": d, "frozen": frozen,
            "bias": bias}


def _rms(kind, N, D, dtype="bf16", wdtype="bf16", rdtype="bf16", q="", group=0):
    """rdtype: the residual's type ('': none); group: columns that share a scale (0: the row)."""
    return {"kind": kind, "N": N, "D": D, "dtype": dtype, "wdtype": wdtype, "rdtype": rdtype, "q": q, "group": group}


def listed():
    return [
        # a policy's gradient over logits that a model returned: two sequences of 2048 tokens, the prompts (40%) masked
        dict(_lp("lp", 4096, 151936, ignored=0.4), name="lp_4096"),
        # a short continuation's rows in fp32: launches count
        dict(_lp("lp", 16, 151936, "fp32", T=0.7), name="lp_16_fp32"),
        # one decoding step of eight sequences: the sampled tokens and twenty alternatives
        dict(_lp("lp_top", 8, 128256, T=0.8, K=20), name="lp_top_8"),
        # a prompt's log-probabilities with five alternatives, GPT-2-sized vocabulary, rows off alignment
        dict(_lp("lp_top", 2047, 50257, K=5, ignored=0.05), name="lp_top_ragged"),
        # fused with the head: one short answer on a small vocabulary
        dict(_lp("lp_linear", 64, 32000, d=896, T=0.9), name="lp_linear_64"),
        # one 2048-token sequence of the 0.5B-parameter benchmark model
        dict(_lp("lp_linear", 2048, 151936, d=896, ignored=0.4), name="lp_linear_2048"),
        # wide hidden, 128k vocabulary: the largest
        dict(_lp("lp_linear", 8192, 128256, d=4096, ignored=0.02), name="lp_linear_8192"),
        # a prompt's log-probabilities with alternatives, from hidden states; bias, a hidden size that is no multiple of 64
        dict(_lp("lp_linear_top", 511, 50257, d=1000, K=20, bias=True), name="lp_linear_top_511"),
        # the norm before the head of the 0.5B-parameter benchmark model, 16384 tokens
        dict(_rms("rms", 16384, 896), name="rms_16384"),
        # a decoding step of eight sequences with an fp32 residual stream
        dict(_rms("rms_eval", 8, 4096, rdtype="fp32"), name="rms_eval_8"),
        # a decoding step of sixteen sequences into e4m3, a scale per 128 columns
        dict(_rms("rms_q", 16, 4096, q="e4m3", group=128), name="rms_q_16"),
        # a batch's hidden states into int8, a scale per token
        dict(_rms("rms_q", 8192, 3584, q="int8"), name="rms_q_8192"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["lp", "lp", "lp_top", "lp_top", "lp_linear", "lp_linear", "lp_linear", "lp_linear_top", "rms",
                       "rms", "rms_eval", "rms_q", "rms_q"])
    if kind.startswith("rms"):
        D = _log(rng, 1, 256) * 64 if rng.random() < 0.6 else _log(rng, 16, 20000)
        N = _log(rng, 1, min(65536, 65536 * 4096 // D))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        case = _rms(kind, N, D, dtype, rng.choice([dtype, "fp32"]), rng.choice([dtype, dtype, "fp32", ""]))
        if kind == "rms_q":
            case.update(q=rng.choice(["e4m3", "int8"]), group=rng.choice([0, 0, 32, 64, 128, 128, 256]))
        return case
    V = _log(rng, 1000, 152064)
    T = rng.choice([1.0, 1.0, 1.0, 0.7, 0.9, 1.5, 3.0])
    ignored = rng.choice([0.0, 0.05, 0.4])
    K = _log(rng, 1, 256) if kind.endswith("top") else 0
    if kind.startswith("lp_linear"):
        # hidden sizes of models are mostly multiples of 64; the head's product is computed in bf16
        d = _log(rng, 2, 64) * 64 if rng.random() < 0.7 else _log(rng, 16, 256) * 8 + 8
        most = 8192 * 4096 * 128256 // (2 * d * V) if kind == "lp_linear" else 4096 * 151936 // (2 * V)
        return _lp(kind, _log(rng, 1, min(16384, most)), V, "bf16", T, K, ignored, d,
                   kind == "lp_linear" and rng.random() < 0.3, rng.random() < 0.2)
    N = _log(rng, 1, min(16384, 4096 * 151936 // (2 * V)))
    return _lp(kind, N, V, rng.choice(["bf16", "bf16", "fp16", "fp32"]), T, K, ignored)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s, dt, N, kind = {"case": case}, DTYPES[case["dtype"]], case["N"], case["kind"]
    if kind.startswith("rms"):
        # hidden states: features of unlike scales, a residual stream larger than what a layer adds; weights near 1
        D = case["D"]
        scales = torch.exp(0.5 * randn(D))
        s["x"] = (randn(N, D) * scales + 0.1).to(dt)
        s["r"] = (randn(N, D) * 3 * scales).to(DTYPES[case["rdtype"]]) if case["rdtype"] else None
        s["w"] = (1 + 0.2 * randn(D)).to(DTYPES[case["wdtype"]])
        if kind == "rms":
            s["dy"] = randn(N, D).to(dt)
            s["ds"] = (0.5 * randn(N, D)).to(DTYPES[case["rdtype"]]) if case["rdtype"] else None
            for name in ("x", "r", "w"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
        return s
    V = case["V"]
    tokens = torch.randint(0, V, (N,), generator=g, device=dev)
    # what a trained model gives its own tokens: up to 12 above the other logits
    likely = 12 * torch.rand(N, 1, generator=g, device=dev)
    if kind == "lp_linear":
        # after a final norm, and a usual initialisation of the head
        d = case["d"]
        w = randn(V, d) * 0.04
        s["h"] = (randn(N, d) + likely / max(0.0016 * d, 0.5) * w[tokens]).to(dt).requires_grad_(True)
        s["w"] = w.to(dt).requires_grad_(not case["frozen"])
        s["b"] = (randn(V) * 0.1).to(dt).requires_grad_(not case["frozen"]) if case["bias"] else None
    elif kind == "lp_linear_top":
        # a head that was held in 8 bits, and hidden states on a grid: every product and sum is exact in 32 bits, so
        # that equal logits are equal for whoever computes them
        s["h"] = (torch.round(randn(N, case["d"]) * 16) / 16).to(dt)
        s["w"] = (torch.round(randn(V, case["d"]) * 24).clamp(-127, 127) / 512).to(dt)
        s["b"] = (torch.round(randn(V) * 16) / 128).to(dt) if case["bias"] else None
    else:
        x = randn(N, V) * 2
        s["x"] = x.scatter_add_(1, tokens[:, None], likely).to(dt).requires_grad_(kind == "lp")
    masked = torch.rand(N, generator=g, device=dev) < case["ignored"]
    masked[0] = False
    s["tokens"] = tokens.masked_fill_(masked, IGNORE)
    if kind in ("lp", "lp_linear"):
        # advantages over the rows that count, and a small weight on the entropy
        n = max(1.0, N * (1 - case["ignored"]))
        s["g"] = randn(N) / n
        s["gh"] = torch.full((N,), 0.01 / n, device=dev) * (1 + 0.1 * randn(N))
    return s


def _lp_rows(case, x, tokens, want_grad, g=None, gh=None):
    """Log-probabilities, entropies and log-softmax of the rows of logits x (32 bits), and the logits' gradient."""
    counts = tokens != IGNORE
    at = torch.where(counts, tokens, 0)[:, None]
    z = (x - x.amax(1, keepdim=True)) / case["T"]
    e = torch.exp(z)
    s = e.sum(1, keepdim=True)
    lp = z - torch.log(s)
    p = e / s
    entropy = -(p * lp).sum(1)
    logprob = lp.gather(1, at)[:, 0]
    out = {"logprobs": torch.where(counts, logprob, 0.0), "entropy": torch.where(counts, entropy, 0.0)}
    if not want_grad:
        return out, lp, counts
    grad = p * (-g[:, None] - gh[:, None] * (lp + entropy[:, None]))
    grad.scatter_add_(1, at, g[:, None])
    return out, grad * (counts / case["T"])[:, None], counts


def _top_rows(case, x, lp, counts):
    """The K largest of each row, the lowest column first among equals; 0 and -1 where the row does not count."""
    at = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["K"]]
    return {"top_logprobs": torch.where(counts[:, None], lp.gather(1, at), 0.0),
            "top_indices": torch.where(counts[:, None], at, -1)}


def _values(q, scale, group, D):
    """What an 8-bit output stands for, in bf16: every e4m3 and int8 number is one of bf16's."""
    out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    q = q.to(torch.bfloat16)
    if not group:
        return torch.mul(q, scale[:, None], out=out)
    if D % group:
        return torch.mul(q, scale.repeat_interleave(group, 1)[:, :D], out=out)
    torch.mul(q.view(-1, D // group, group), scale[:, :, None], out=out.view(-1, D // group, group))
    return out


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind.startswith("rms"):
        out, D = {}, case["D"]
        x, w = s["x"].float(), s["w"].float()
        if s["r"] is not None:
            out["s"] = (x + s["r"].float()).to(s["r"].dtype)
            x = out["s"].float()
        r = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
        n = x * r
        y = n * w
        if kind == "rms_q":
            most, group = LARGEST[case["q"]], case["group"] or D
            a = torch.nn.functional.pad(y.abs(), (0, -D % group)).view(case["N"], -1, group).amax(2)
            scale = a.clamp(min=1e-30) / most
            v = y / scale.repeat_interleave(group, 1)[:, :D]
            q = (torch.round(v) if case["q"] == "int8" else v).to(DTYPES[case["q"]])
            scale = scale if case["group"] else scale[:, 0]
            return {**out, "values": _values(q, scale, case["group"], D), "scales": scale}
        out["y"] = y.to(s["x"].dtype)
        if kind == "rms_eval":
            return out
        dy = s["dy"].float()
        a = dy * w
        dx = r * (a - n * (a * n).mean(1, keepdim=True))
        if s["ds"] is not None:
            dx = dx + s["ds"].float()
            out["dr"] = dx.to(s["r"].dtype)
        out["dx"] = dx.to(s["x"].dtype)
        out["dw"] = (dy * n).sum(0).to(s["w"].dtype)
        return out
    if kind in ("lp", "lp_top"):
        x = s["x"].float()
    else:
        h, w = s["h"].float(), s["w"].float()
        x = h @ w.t()
        if s["b"] is not None:
            x = x + s["b"].float()
    if kind.endswith("top"):
        out, lp, counts = _lp_rows(case, x, s["tokens"], False)
        return {**out, **_top_rows(case, x, lp, counts)}
    out, grad, _ = _lp_rows(case, x, s["tokens"], True, s["g"], s["gh"])
    if kind == "lp":
        return {**out, "dx": grad.to(s["x"].dtype)}
    out["dh"] = (grad @ w).to(s["h"].dtype)
    if not case["frozen"]:
        out["dw"] = (grad.t() @ h).to(s["w"].dtype)
        if s["b"] is not None:
            out["db"] = grad.sum(0).to(s["b"].dtype)
    return out


def _own(s):
    from chronicals_amd.kernels.rms_norm import rms_norm, rms_norm_quantized
    from chronicals_amd.kernels.token_logprobs import linear_token_logprobs, token_logprobs

    case = s["case"]
    kind = case["kind"]
    if kind == "rms_q":
        q, scale, *kept = rms_norm_quantized(s["x"], s["w"], s["r"], EPS, DTYPES[case["q"]], case["group"] or None)
        out = {"values": _values(q, scale, case["group"], case["D"]), "scales": scale}
        return {**out, "s": kept[0]} if kept else out
    if kind == "rms_eval":
        with torch.no_grad():
            y = rms_norm(s["x"], s["w"], s["r"], EPS)
        return {"y": y} if s["r"] is None else {"y": y[0], "s": y[1]}
    if kind == "rms":
        leaves = {"dx": s["x"], "dw": s["w"]}
        y = rms_norm(s["x"], s["w"], s["r"], EPS)
        if s["r"] is None:
            return {"y": y.detach(), **dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), s["dy"])))}
        leaves["dr"] = s["r"]
        grads = torch.autograd.grad(y, list(leaves.values()), (s["dy"], s["ds"]))
        return {"y": y[0].detach(), "s": y[1].detach(), **dict(zip(leaves, grads))}
    how = {"temperature": case["T"], "top_k": case["K"]}
    if kind.endswith("top"):
        with torch.no_grad():
            if kind == "lp_top":
                out = token_logprobs(s["x"], s["tokens"], **how)
            else:
                out = linear_token_logprobs(s["h"], s["w"], s["tokens"], s["b"], **how)
        return out._asdict()
    if kind == "lp":
        out = token_logprobs(s["x"], s["tokens"], **how)
        leaves = {"dx": s["x"]}
    else:
        out = linear_token_logprobs(s["h"], s["w"], s["tokens"], s["b"], **how)
        leaves = {"dh": s["h"]}
        if not case["frozen"]:
            leaves["dw"] = s["w"]
            if s["b"] is not None:
                leaves["db"] = s["b"]
    grads = torch.autograd.grad((out.logprobs, out.entropy), list(leaves.values()), (s["g"], s["gh"]))
    return {"logprobs": out.logprobs.detach(), "entropy": out.entropy.detach(), **dict(zip(leaves, grads))}


def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return _plain(s)


def work(case):
    """Each input read once and each output written once; the products over the rows that count."""
    kind, N, size = case["kind"], case["N"], SIZE[case["dtype"]]
    if kind.startswith("rms"):
        D = case["D"]
        rsize = SIZE[case["rdtype"]] if case["rdtype"] else 0
        params = D * SIZE[case["wdtype"]]
        read, written = size + rsize, rsize + (SIZE[case["q"]] if kind == "rms_q" else size)
        if kind == "rms_q":
            scales = 4 * N * (-(-D // case["group"]) if case["group"] else 1)
            return {"bytes": N * D * (read + written) + params + scales, "flops": 8 * N * D}
        if kind == "rms_eval":
            return {"bytes": N * D * (read + written) + params, "flops": 6 * N * D}
        # the gradients of y and s come in, those of x and (of another type) of the residual go out
        more = size + rsize + size + (rsize if case["rdtype"] != case["dtype"] else 0)
        return {"bytes": N * D * (read + written + more) + 2 * params, "flops": 18 * N * D}
    V, K = case["V"], case["K"]
    live = N * (1.0 - case["ignored"])
    rows = 16 * N + 12 * N * K
    if kind == "lp_top":
        return {"bytes": int(live * V * size + rows), "flops": int(6 * live * V)}
    if kind == "lp":
        return {"bytes": int((live + N) * V * size + rows + 8 * N), "flops": int(12 * live * V)}
    d = case["d"]
    read, written, products = (live * d + V * d) * size, 0, 1
    if kind == "lp_linear":
        products, written = 2, N * d * size
        if not case["frozen"]:
            products, written = 3, written + V * d * size + (V * size if case["bias"] else 0)
    return {"bytes": int(read + written + rows), "flops": int(2 * products * live * d * V)}


def _e4m3(v):
    """v rounded to e4m3 in 64 bits: three bits behind the leading one, steps of 2^-9 below 2^-6, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    kind, N = case["kind"], case["N"]
    if kind.startswith("rms"):
        out, D = {}, case["D"]
        x, w = s["x"].detach().double(), s["w"].detach().double()
        if s["r"] is not None:
            # what is kept, and normalised, is the sum as its type holds it
            out["s"] = (x + s["r"].detach().double()).to(s["r"].dtype).double()
            x = out["s"]
        norm = torch.linalg.vector_norm(x, dim=1, keepdim=True)
        root = torch.sqrt(norm * norm / D + EPS)
        y = x / root * w
        if kind == "rms_q":
            most, group = LARGEST[case["q"]], case["group"] or D
            groups = torch.zeros(N, -(-D // group) * group, dtype=torch.float64, device=x.device)
            groups[:, :D] = y
            groups = groups.view(N, -1, group)
            scale = groups.abs().max(2).values.clamp(min=1e-30) / most
            v = groups / scale[:, :, None]
            v = torch.round(v) if case["q"] == "int8" else _e4m3(v)
            out["values"] = (v * scale[:, :, None]).view(N, -1)[:, :D].contiguous()
            out["scales"] = scale if case["group"] else scale[:, 0].contiguous()
            return out
        out["y"] = y
        if kind == "rms_eval":
            return out
        dy = s["dy"].double()
        a, n = dy * w, x / root
        # the projection of dy * w off the normalised row
        dx = (a - n * ((a * n).sum(1, keepdim=True) / D)) / root
        if s["ds"] is not None:
            dx = dx + s["ds"].double()
            out["dr"] = dx
        return {**out, "dx": dx, "dw": torch.einsum("nd,nd->d", dy, n)}
    V, T, K, tokens = case["V"], case["T"], case["K"], s["tokens"]
    if N * V > 1 << 31:
        return None
    linear, grads = kind.startswith("lp_linear"), kind in ("lp", "lp_linear")
    counts = tokens != IGNORE
    dev = tokens.device
    out = {"logprobs": torch.zeros(N, dtype=torch.float64, device=dev),
           "entropy": torch.zeros(N, dtype=torch.float64, device=dev)}
    if linear:
        h, w = s["h"].detach().double(), s["w"].detach().double()
        if grads:
            out["dh"] = torch.zeros_like(h)
            if not case["frozen"]:
                out["dw"] = torch.zeros_like(w)
                if s["b"] is not None:
                    out["db"] = torch.zeros(V, dtype=torch.float64, device=dev)
    elif grads:
        out["dx"] = torch.empty(N, V, dtype=torch.float64, device=dev)
    if K:
        out["top_logprobs"] = torch.zeros(N, K, dtype=torch.float64, device=dev)
        out["top_indices"] = torch.full((N, K), -1, device=dev)
    for a in range(0, N, 2048):
        r = slice(a, min(a + 2048, N))
        if linear:
            x = h[r] @ w.t()
            if s["b"] is not None:
                x += s["b"].detach().double()
        else:
            x = s["x"][r].detach().double()
        c = counts[r]
        lp = torch.log_softmax(x / T, 1)
        p = lp.exp()
        entropy = -torch.xlogy(p, p).sum(1)
        tok = tokens[r].clamp(min=0)[:, None]
        out["logprobs"][r] = lp.gather(1, tok)[:, 0] * c
        out["entropy"][r] = entropy * c
        if K:
            # by value, then the lower column: the values are distinct from their neighbours by far more than 2^-40
            at = (x - torch.arange(V, device=dev) * 2.0 ** -40).topk(K, 1).indices
            out["top_logprobs"][r] = lp.gather(1, at) * c[:, None]
            out["top_indices"][r] = torch.where(c[:, None], at, -1)
        if not grads:
            continue
        g, gh = (s[k][r].double()[:, None] for k in ("g", "gh"))
        grad = lp.add_(entropy[:, None]).mul_(-gh).sub_(g).mul_(p)
        grad.scatter_add_(1, tok, g)
        grad *= c[:, None] / T
        if not linear:
            out["dx"][r] = grad
            continue
        out["dh"][r] = grad @ w
        if not case["frozen"]:
            out["dw"].addmm_(grad.t(), h[r])
            if s["b"] is not None:
                out["db"] += grad.sum(0)
    return out
