"""Plain float64 forms of attention's windows and trees (as which pairs are allowed, for ``layer_oracle.attention``) and of
tokens' log probabilities with their gradient, and the error bounds that the kernels' float32 arithmetic gives."""
from __future__ import annotations

import math

import torch

from layer_oracle import EPS32, TINY, U


def window_allowed(queries, keys, lengths, batch, offset, window, sinks):
    """[batch, queries, keys] booleans; ``offset`` None: the queries are the sequence's last tokens."""
    out = torch.zeros(batch, queries, keys, dtype=torch.bool)
    for b in range(batch):
        n = keys if lengths is None else int(lengths[b])
        off = n - queries if offset is None else offset
        p, j = torch.arange(queries).view(-1, 1) + off, torch.arange(keys).view(1, -1)
        out[b] = (j < n) & (j <= p) & ((p - j < window) | (j < sinks))
    return out


def tree_allowed(parents, keys, lengths, batch):
    """[batch, nodes, keys] booleans from parents [batch][nodes]."""
    nodes = len(parents[0])
    out = torch.zeros(batch, nodes, keys, dtype=torch.bool)
    for b in range(batch):
        n = keys if lengths is None else int(lengths[b])
        for i in range(nodes):
            out[b, i, :max(0, n - nodes)] = True
            at = i
            while True:
                if n - nodes + at >= 0:
                    out[b, i, n - nodes + at] = True
                if not 0 <= parents[b][at] < at:
                    break
                at = parents[b][at]
    return out


def log_probs(z, tokens, g=None, gh=None, gtop=None, top=0):
    """Results in float64 for ``z`` [rows, vocab], ``tokens`` [rows, each], and for each a bound on a float32 evaluation's
    error: ``(values, bounds)`` by name.

    With d = z - max z, an exponential is off by 3 |d| + 4 units of float32 roundoff u (the difference, its product with
    log2(e), the instruction), sums of n values by n + 48 (a thread adds a 256th of them, then the joins and rescalings),
    a logarithm by 3 of its value and one absolute, a difference by one of each operand.
    """
    z = z.double()
    rows, vocab = z.shape
    u = EPS32
    m = z.max(1, keepdim=True).values
    empty = (m == -math.inf).squeeze(1)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    d = z - m
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(torch.where(total > 0, total, torch.ones_like(total)))
    # not z - (m + log_total): of rows at float32's lowest value the sum would lose the logarithm in 64 bits, too
    lp = torch.where(empty.unsqueeze(1), torch.full_like(z, -math.inf), d - log_total)
    p = torch.exp(lp)
    n = vocab / 256 + 48
    ad = torch.where(p > 0, d.abs(), torch.zeros_like(d))
    mean_d = (p * ad).sum(1, keepdim=True)
    rel = u * (n + 4 + 3 * mean_d)                    # of the sum
    log_err = rel + u * (3 * log_total.abs() + 2)     # of its logarithm
    lp_err = log_err + u * (2 * d.abs() + 2 * torch.where(lp.isinf(), torch.zeros_like(lp), lp.abs()))
    asked = (tokens >= 0) & (tokens < vocab)
    at = torch.where(asked, tokens, torch.zeros_like(tokens))
    got = torch.gather(lp, 1, at)
    got = torch.where(asked, got, torch.where(tokens < 0, 0.0, math.nan).double())
    res = {"log_probs": got, "log_probs_err": torch.gather(lp_err, 1, at)}
    h = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
    h_err = (log_err + (p * ad * u * (3 * ad + 5 + n)).sum(1, keepdim=True) + mean_d * (rel + 2 * u)).squeeze(1) + u * h.abs()
    res["entropy"], res["entropy_err"] = h, h_err
    if top:
        # the lowest of equal ones first; NaN before all
        values, order = torch.sort(z, dim=1, descending=True, stable=True)
        res["top_tokens"] = order[:, :top]
        res["top_log_probs"] = torch.gather(lp, 1, order[:, :top])
        res["top_log_probs_err"] = torch.gather(lp_err, 1, order[:, :top])
    if g is None and gh is None and gtop is None:
        return res
    given = torch.zeros_like(z)
    size = torch.zeros_like(z)
    sums = torch.zeros(rows, 1, dtype=torch.float64)
    sizes = torch.zeros(rows, 1, dtype=torch.float64)
    for idx, grad, ok in ((tokens, g, asked), (res.get("top_tokens"), gtop, None)):
        if grad is None:
            continue
        grad = grad.double() if ok is None else torch.where(ok, grad.double(), torch.zeros((), dtype=torch.float64))
        where = idx if ok is None else at
        given.scatter_add_(1, where, grad)
        size.scatter_add_(1, where, grad.abs())
        sums += grad.sum(1, keepdim=True)
        sizes += grad.abs().sum(1, keepdim=True)
    terms = tokens.shape[1] + top + 4
    slope = -sums
    slope_err = u * terms * sizes
    if gh is not None:
        gh = gh.double().unsqueeze(1)
        inner = torch.where(p > 0, lp + h.unsqueeze(1), torch.zeros_like(p))
        slope = slope - gh * inner
        lp_off = torch.where(p > 0, lp_err, torch.zeros_like(p))
        slope_err = slope_err + gh.abs() * (lp_off + h_err.unsqueeze(1) + 3 * u * inner.abs())
    dz = p * slope + given
    # p = exp(lp) of an lp that is off by lp_err, and of the exponential's own rounding
    # below 2^-126 the exponential gives 0
    some = p > 0
    p_err = torch.where(some, p * (lp_err + u * (2 * lp.abs() + 4)) + 2.0 ** -126, torch.zeros_like(p))
    slope_err = torch.where(some, slope_err, torch.zeros_like(p))
    err = p_err * slope.abs() + p * slope_err + u * terms * size + u * dz.abs() * 4
    zero = empty.unsqueeze(1)
    res["grad"] = torch.where(zero, torch.zeros_like(dz), dz)
    res["grad_err"] = torch.where(zero, torch.zeros_like(err), err)
    return res


def rounded_bound(res, name, dtype):
    """The bound of a float32 result rounded to ``dtype``."""
    return res[name + "_err"] * (1 + U[dtype]) + U[dtype] * res[name].abs() + TINY[dtype]
