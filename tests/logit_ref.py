"""Plain 64-bit forms of the log probabilities and of distillation, on the CPU, with the bounds of
what fp32 arithmetic may be off by.

Counted, in units of E32 = 2^-24, for x = z / tau, d = x - max x:
  an exponent: the difference, 1 / tau, the product: 3 |d|; an exponential 2 more
  a row's sum: the exponentials' errors weighted with p, no lane adding more than
    max(64, V / 256) in sequence, 64 more for joining lanes
  a logarithm 3 of its value, a product or a sum 1
Exponentials below 2^-126 are zero."""

import math

import torch

from train_ref import E32, TINY, U

F64 = torch.float64


def _z0(t):
    return torch.nan_to_num(t, 0.0, 0.0, 0.0)


class Softmax:
    """p, log p and statistics of z / tau in float64; bounds of sums (rho) and log p (lp_err)."""

    def __init__(self, z, tau=1.0, keep=None):
        """keep: the classes that count (the rest of a list), all by default."""
        x = z.double() / tau
        if keep is not None:
            x = torch.where(keep, x, -torch.inf)
        v = x.shape[-1]
        self.x = x
        self.m = x.amax(-1, keepdim=True)
        # from differences: a row of the lowest fp32 value has no digits left for its log s
        self.gap = self.m - x
        self.log_s = torch.logsumexp(-self.gap, -1, keepdim=True)
        self.lse = self.m + self.log_s
        self.log_p = -self.gap - self.log_s
        # what lies half a last place beyond the largest fp32 value rounds to an infinity
        self.log_p = torch.where(self.log_p <= -(2.0 ** 128 - 2.0 ** 103), -torch.inf, self.log_p)
        self.p = torch.exp(self.log_p)
        pd = _z0(self.p * self.gap)
        self.d1 = pd.sum(-1, keepdim=True)
        self.d2 = _z0(pd * self.gap).sum(-1, keepdim=True)
        self.chain = max(64, v // 256) + 64
        self.rho = (self.chain + 4 * self.d1 + 4) * E32
        self.lp_err = self.rho + 4 * E32 * (_z0(self.gap) + _z0(self.log_s)) \
            + E32 * _z0(self.log_p).abs()
        self.h = -_z0(self.p * self.log_p).sum(-1, keepdim=True)
        self.h_err = self.rho + 1e-30 + E32 * (4 * _z0(self.log_s) + 2 * self.h + 4 * self.d2
                                               + (self.chain + 12) * self.d1) + self.rho * self.d1
        # of p, and of p times (log p + h)
        self.p_err = self.p * (self.rho + (3 * _z0(self.gap) + 6) * E32) + 1e-37


def top(z, k):
    """The k largest classes of each row, ties by the lower class."""
    return torch.sort(z.double(), dim=-1, descending=True, stable=True)[1][..., :k]


def log_probs(z, y=None, k=0, tau=1.0, ignore=-100):
    """{name: (value, bound)} of the outputs, and the top classes."""
    s = Softmax(z, tau)
    live = torch.ones(z.shape[:-1], dtype=torch.bool) if y is None else y != ignore
    zero = torch.zeros((), dtype=F64)
    out = {}
    if y is not None:
        inside = (y >= 0) & (y < z.shape[-1])
        at = torch.where(inside, y, 0).long()[..., None]
        lp = torch.where(inside, s.log_p.gather(-1, at)[..., 0], torch.nan)
        out["log_probs"] = (torch.where(live, lp, zero), s.lp_err.gather(-1, at)[..., 0])
    h = torch.where(torch.isfinite(s.lse), s.h, torch.nan)[..., 0]
    out["entropy"] = (torch.where(live, h, zero), s.h_err[..., 0])
    ids = None
    if k:
        ids = top(z, k)
        out["top_log_probs"] = (torch.where(live[..., None], s.log_p.gather(-1, ids), zero),
                                s.lp_err.gather(-1, ids))
        ids = torch.where(live[..., None], ids, ignore)
    return out, ids


def log_probs_grad(z, y, ids, gy, gh, gt, tau, dtype, ignore=-100):
    """(gradient, bound); gy, gh, gt: the outputs' gradients, or None."""
    s = Softmax(z, tau)
    n = torch.zeros(z.shape[:-1], dtype=F64)
    live = torch.ones(z.shape[:-1], dtype=torch.bool) if y is None else y != ignore
    push, size, delta = n[..., None].clone(), n[..., None].clone(), torch.zeros_like(s.x)
    weight = torch.zeros_like(s.x)
    for at, g in (((None if y is None else y[..., None]), None if gy is None else gy[..., None]),
                  (ids, gt)):
        if g is None:
            continue
        g = g.double()
        push, size = push + g.sum(-1, keepdim=True), size + g.abs().sum(-1, keepdim=True)
        at = torch.where(live[..., None], at, 0).long()
        delta.scatter_add_(-1, at, g)
        weight.scatter_add_(-1, at, g.abs())
    gh = n[..., None] if gh is None else gh.double()[..., None]
    log_p = _z0(s.log_p) * (s.p > 0)
    want = delta - s.p * push - gh * s.p * (log_p + s.h)
    gap = _z0(s.gap) * (s.p > 0)
    size = size + gh.abs() * (log_p.abs() + s.h)
    err = s.p_err * size + s.p * (30 * E32 * size
                                  + gh.abs() * (s.h_err + s.rho
                                                + 10 * E32 * (s.h + _z0(s.log_s) + gap)))
    err = (1.1 * err + 6 * E32 * (weight + s.p * size)) / tau
    want = torch.where(live[..., None], want / tau, torch.zeros((), dtype=F64))
    return want, err + 1.01 * U[dtype] * want.abs() + TINY[dtype]


class Distill:
    """Row losses and gradients (for a loss's gradient of 1) with their bounds."""

    def __init__(self, z, ids, t, tau=1.0, rest=False, ignore=-100):
        v, k = z.shape[-1], ids.shape[-1]
        s = Softmax(z, tau)
        zero = torch.zeros((), dtype=F64)
        some = ids != ignore
        self.live = some[..., 0]
        bad = (some & ((ids < 0) | (ids >= v))).any(-1)
        inside = some & (ids >= 0) & (ids < v)
        at = torch.where(inside, ids, 0).long()
        t = torch.where(inside, t.double(), -torch.inf)
        if rest:
            q, log_q = torch.exp(t), t
            lq_err, eq = torch.zeros_like(q), (2 * _z0(t.abs()) + 3) * E32
        else:
            log_q = t - torch.logsumexp(t, -1, keepdim=True)
            q = torch.exp(log_q)
            depth = _z0(t.amax(-1, keepdim=True) - t)
            sums = (k + 8 + 4 * (q * depth).sum(-1, keepdim=True)) * E32
            lq_err = sums + 4 * E32 * (depth + _z0(log_q).abs())
            eq = sums + (3 * depth + 5) * E32
        q = torch.where(inside, q, zero)
        log_p = s.log_p.gather(-1, at)
        terms = torch.where(q != 0, q * (log_q - log_p), zero)
        loss = terms.sum(-1)
        size = torch.where(q != 0, q * (log_q.abs() + log_p.abs()), zero)
        err = (_z0(q) * (lq_err + s.lp_err.gather(-1, at)) + _z0(q * eq * (log_q - log_p).abs())
               + 3 * E32 * _z0(size)).sum(-1) + k * E32 * _z0(terms.abs()).sum(-1)
        w = q.sum(-1, keepdim=True)
        if rest:
            listed = torch.zeros((*z.shape[:-1], v + 1), dtype=torch.bool)
            listed.scatter_(-1, torch.where(inside, ids, v).long(), True)
            o = Softmax(z, tau, ~listed[..., :v])
            others = o.m != -torch.inf      # no class outside the list: nothing to leave it
            left = torch.where(others, torch.clamp(1.0 - w, min=0.0), zero)
            w = torch.where(others, torch.clamp(w, min=1.0), torch.where(w != 0, w, torch.nan))
        dense = torch.zeros_like(s.x).scatter_add_(-1, at, q)
        dense_err = torch.zeros_like(s.x).scatter_add_(-1, at, _z0(q * eq))
        dz = w * s.p - dense
        # w itself is off where the list sums to more than 1
        w_err = _z0(q * eq).sum(-1, keepdim=True) + (k + 8) * E32
        dz_err = w * s.p_err + s.p * w_err + dense_err + 6 * E32 * (w * s.p + _z0(dense))
        if rest:
            log_r = (o.m - s.m) + (o.log_s - s.log_s)   # -inf where nothing is left
            log_r = torch.where(torch.isfinite(o.m), log_r, -torch.inf)
            part = torch.where(left != 0, left * (torch.log(left) - log_r), zero)[..., 0]
            loss = loss + part
            # up to the list's own rounding, a rest counts as none
            left_err = torch.where(others, w_err + (8 + 2 * math.log(k)) * E32, zero)
            log_left = torch.where(left > 0, torch.log(left), zero)
            err = err + (left_err * (_z0(log_left - log_r).abs() + 1)
                         + left * (o.rho + s.rho + 4 * E32 * (
                             _z0(o.m - s.m).abs() + _z0(o.log_s) + _z0(s.log_s)
                             + log_left.abs())))[..., 0] + 3 * E32 * _z0(part.abs())
            r = _z0(o.p)
            dz = dz - left * r
            dz_err = dz_err + r * left_err + left * (_z0(o.p_err)) + 6 * E32 * left * r
        nan = bad | ~torch.isfinite(s.lse[..., 0]) | torch.isnan(w[..., 0])
        self.loss = torch.where(self.live, torch.where(nan, torch.nan, loss * tau ** 2), zero)
        self.loss_err = 1.1 * _z0(err) * tau ** 2 + 4 * E32 * _z0(self.loss).abs()
        dz = torch.where(nan[..., None], torch.nan, dz * tau)
        self.dz = torch.where(self.live[..., None], dz, zero)
        self.dz_err = 1.1 * _z0(dz_err) * tau

    def mean(self):
        n = int(self.live.sum())
        rows = self.loss.numel()
        return (self.loss.sum() / n, self.loss_err[self.live].sum() / n
                + (rows / 64 + 20) * E32 * self.loss.abs().sum() / n, n)

    def grad_bound(self, g, dtype):
        want = self.dz * g
        return want, (self.dz_err + 4 * E32 * _z0(self.dz).abs()) * abs(g) \
            + 1.01 * U[dtype] * _z0(want).abs() + TINY[dtype]
