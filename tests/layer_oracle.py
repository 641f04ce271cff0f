"""Plain float64 layer norm, attention and GELU with their gradients, and the error bounds that the
kernels' arithmetic gives: what a float32 (or, for operands, 16-bit) evaluation may be off by, from the
rounding errors of its steps.  ``U[dtype]`` is a type's unit roundoff."""
from __future__ import annotations

import math

import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}  # half a subnormal step or less
EPS32 = 2.0 ** -24


def layer_norm(h, w, b, eps, dy=None, dh=None):
    """(y, dx, dw, db) in float64 and elementwise bounds' absolute parts (see test)."""
    h, w = h.double(), w.double()
    f = h.shape[-1]
    mean = h.mean(-1, keepdim=True)
    c = h - mean
    rstd = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    n = c * rstd
    y = n * w + (0 if b is None else b.double())
    if dy is None:
        return y, n, rstd
    dy = dy.double()
    a = dy * w
    dx = rstd * (a - a.mean(-1, keepdim=True) - n * (a * n).mean(-1, keepdim=True))
    if dh is not None:
        dx = dx + dh.double()
    return y, dx, (dy * n).reshape(-1, f).sum(0), dy.reshape(-1, f).sum(0)


def allowed(queries, keys, lengths, batch, causal, offset):
    """[batch, queries, keys] booleans; ``offset`` None: the queries are the sequence's last tokens."""
    out = torch.zeros(batch, queries, keys, dtype=torch.bool)
    for b in range(batch):
        n = keys if lengths is None else int(lengths[b])
        j = torch.arange(keys).view(1, -1)
        ok = (j < n).expand(queries, keys)
        if causal:
            off = n - queries if offset is None else offset
            ok = ok & (j <= torch.arange(queries).view(-1, 1) + off)
        out[b] = ok
    return out


def attention(q, k, v, scale, ok, do=None):
    """Output, log sums and gradients in float64, with a bound for each on a kernel's error per unit of
    relative error: what a relative error of one in every product's operands would come to.  Keys that are
    never allowed may hold anything."""
    b, h, t, d = q.shape
    hk = k.shape[1]
    g = h // hk
    seen = ok.any(1).view(b, 1, -1, 1)
    zero = torch.zeros((), dtype=torch.float64)
    k = torch.where(seen, k.double(), zero).repeat_interleave(g, 1)
    v = torch.where(seen, v.double(), zero).repeat_interleave(g, 1)
    some = ok.any(2).view(b, 1, t, 1)
    q = torch.where(some, q.double(), zero)
    ok = ok.unsqueeze(1)
    s = (q @ k.transpose(2, 3)) * scale
    size = (q.abs() @ k.abs().transpose(2, 3)) * scale  # of the terms of a score
    s = s.masked_fill(~ok, -math.inf)
    lse = torch.logsumexp(s, -1, keepdim=True)
    p = torch.where(ok, torch.exp(s - torch.where(lse.isinf(), zero, lse)), zero)
    o = p @ v
    # a score's error, in units of float32 roundoff: d + 8 roundings of its terms
    worst = torch.where(ok, size, zero).amax(-1, keepdim=True)
    gamma = (d + 8) * EPS32 * (1 + 2 * worst)
    res = {"o": o, "lse": lse.squeeze(-1), "gamma": gamma, "o_terms": p @ v.abs()}
    if do is None:
        return res
    do = torch.where(some, do.double(), zero)
    dp = do @ v.transpose(2, 3)
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    spread = p * (do.abs() @ v.abs().transpose(2, 3) + (do.abs() * o.abs()).sum(-1, keepdim=True))

    def heads(x):
        return x.view(b, hk, g, *x.shape[2:]).sum(2)

    res["dq"], res["dq_terms"] = scale * (ds @ k), scale * (spread @ k.abs())
    res["dk"] = heads(scale * (ds.transpose(2, 3) @ q))
    res["dk_terms"] = heads(scale * (spread.transpose(2, 3) @ q.abs()))
    res["dv"] = heads(p.transpose(2, 3) @ do)
    res["dv_terms"] = heads(p.transpose(2, 3) @ do.abs())
    res["gamma_all"] = gamma.max().item()
    return res


def gelu(z, approximate):
    """(value, slope) in float64."""
    z = z.double()
    if approximate == "tanh":
        c = 2 * math.sqrt(2 / math.pi)
        s = torch.sigmoid(c * (z + 0.044715 * z ** 3))
        return z * s, s + z * s * (1 - s) * c * (1 + 3 * 0.044715 * z * z)
    phi = 0.5 * torch.erfc(-z / math.sqrt(2.0))
    return z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def checkpoint8(z):
    """(codes, scales) of float32 rows ``z`` by the definition, in float32 on the CPU."""
    rows, f = z.shape
    groups = -(-f // 128)
    zp = torch.zeros(rows, groups * 128)
    zp[:, :f] = z
    zg = zp.view(rows, groups, 128)
    scale = zg.abs().amax(-1) * torch.tensor(1.0 / 127.0, dtype=torch.float32)
    inv = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
    codes = torch.round(zg * inv.unsqueeze(-1)).to(torch.int8)
    return codes.view(rows, -1)[:, :f], scale
