"""References in 64 bits and tolerances of the token log-probability tests."""
import math

import torch

from tests.distill_common import EXP_ERR, EXP_LEAST, IGNORE


def tokens(g, N, V, ignored=0.2):
    t = torch.randint(0, V, (N,), generator=g)
    t[torch.rand(N, generator=g) < ignored] = IGNORE
    return t


class Reference:
    """Log-probabilities, entropies and the logits' gradient of logits x [N, V] in 64 bits, for gradients g and h of the
    two; and the magnitudes of what they are sums of."""

    def __init__(self, x, tok, T=1.0, g=None, h=None):
        x = x.double()
        N, V = x.shape
        g = torch.zeros(N).double() if g is None else g.double()
        h = torch.zeros(N).double() if h is None else h.double()
        self.T, self.V = T, V
        self.counts = tok != IGNORE
        self.logprobs, self.entropy = torch.zeros(N).double(), torch.zeros(N).double()
        self.size = torch.zeros(N).double()  # what the roundings of a row's sums are relative to
        self.grad, self.mag, self.row_log_softmax = (torch.zeros(N, V).double() for _ in range(3))
        for n in range(N):
            if not self.counts[n]:
                continue
            t = int(tok[n])
            has = 0 <= t < V
            if bool((x[n] == -math.inf).all()):
                self.row_log_softmax[n] = -math.inf
                self.logprobs[n] = -math.inf if has else 0.0
                continue
            lp = torch.log_softmax(x[n] / T, 0)
            p = lp.exp()
            H = -torch.special.xlogy(p, p).sum()
            self.row_log_softmax[n] = lp
            self.logprobs[n] = lp[t] if has else 0.0
            self.entropy[n] = H
            self.size[n] = 1 + abs(float(lp.max())) + H + (abs(float(lp[t])) if has and lp[t] > -math.inf else 0.0)
            low = torch.where(p > 0, lp, 0.0)
            gn = g[n] if has else 0.0
            self.grad[n] = p * (-gn - h[n] * (low + H)) / T
            self.mag[n] = p * (abs(gn) + h[n].abs() * (low.abs() + H + 1)) / T
            if has:
                self.grad[n, t] += gn / T
                self.mag[n, t] += abs(gn) / T
        # The exponentials that a sum is made of are each off by (8 + 4 |u|) 2^-24 with the
        # exponent u in base 2; weighted with themselves |u| is at most log2(V) < 18 in the
        # mean.  Up to V / 256 and a few more additions follow one another; the logarithm
        # and the last operations add a few roundings of the parts.
        self.tol = (128 + V / 256) * 2.0 ** -23 * self.size
        self.grad_tol = 2 * EXP_ERR * self.mag + EXP_LEAST * ((g.abs() + h.abs() * (1000 + self.entropy)) / T)[:, None]

    def top(self, x, k):
        """Log-probabilities and columns of the k largest of each row of x."""
        s = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :k]
        v = self.row_log_softmax.gather(1, s)
        c = self.counts[:, None]
        return torch.where(c, v, 0.0), torch.where(c, s, -1)
