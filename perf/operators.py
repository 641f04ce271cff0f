"""The operators between a transformer block's generated linears, as workloads for measurement.

Three operators, each through the package's public entry points:

``norm``    layer norm over the features, with or without the residual stream's addition before it:
            forward for serving, forward and backward for training
``attend``  attention: a prompt's forward, a training step that recomputes the probabilities in its
            backward pass, and new tokens over a cache of keys and values
``gelu``    GELU whose input is kept in 8 bits: forward for serving; for training also the activation
            computed again from the checkpoint and the backward pass

``own`` chooses between the framework's operators and the same mathematics in elementary torch
operations in float32.  ``exact()`` restates each of them in float64.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda"
EPS = 1e-5
GROUP = 128  # features that share a scale of the 8-bit checkpoint


def listed():
    return [
        # The norm before a block's attention at one decoded token of GPT-2 small: the smallest call.
        {"name": "norm_bf16_token", "kind": "norm", "dtype": "bf16", "weight": "bf16", "rows": 1, "features": 768,
         "bias": True, "residual": True, "step": False},
        # The same in training on 8 sequences of 1024 tokens, float32 weights beside bfloat16 activations.
        {"name": "norm_step_bf16_8k", "kind": "norm", "dtype": "bf16", "weight": "f32", "rows": 8192, "features": 768,
         "bias": True, "residual": True, "step": True},
        # A float32 training step on a ragged batch of wide rows without a bias.
        {"name": "norm_step_f32_wide", "kind": "norm", "dtype": "f32", "weight": "f32", "rows": 1021, "features": 3072,
         "bias": False, "residual": False, "step": True},
        # Prefill of 8 sequences of 1024 tokens through GPT-2 small's attention.
        {"name": "prefill_bf16_8x1024", "kind": "attend", "form": "packed", "dtype": "bf16", "batch": 8, "queries": 1024,
         "keys": 1024, "heads": 12, "kv_heads": 12, "dim": 64, "causal": True, "ragged": False, "step": False},
        # A training step of the same attention.
        {"name": "attend_step_bf16_8x1024", "kind": "attend", "form": "packed", "dtype": "bf16", "batch": 8,
         "queries": 1024, "keys": 1024, "heads": 12, "kv_heads": 12, "dim": 64, "causal": True, "ragged": False,
         "step": True},
        # A float32 training step on short sequences (a check of numerics, a small model).
        {"name": "attend_step_f32_4x512", "kind": "attend", "form": "packed", "dtype": "f32", "batch": 4, "queries": 512,
         "keys": 512, "heads": 12, "kv_heads": 12, "dim": 64, "causal": True, "ragged": False, "step": True},
        # A training step over padded sequences of other lengths than the queries', one of them empty,
        # with key heads shared by three query heads and a head size that fills no tile.
        {"name": "attend_step_f16_ragged", "kind": "attend", "form": "heads", "dtype": "f16", "batch": 6, "queries": 515,
         "keys": 1531, "heads": 12, "kv_heads": 4, "dim": 80, "causal": False, "ragged": True, "step": True},
        # One long prompt, key heads shared by four query heads: the most work of all.
        {"name": "prefill_bf16_1x8192", "kind": "attend", "form": "heads", "dtype": "bf16", "batch": 1, "queries": 8192,
         "keys": 8192, "heads": 16, "kv_heads": 4, "dim": 128, "causal": True, "ragged": False, "step": False},
        # Decoding 64 sequences of different lengths over GPT-2 small's cache, one token each.
        {"name": "decode_bf16_64", "kind": "attend", "form": "heads", "dtype": "bf16", "batch": 64, "queries": 1,
         "keys": 1024, "heads": 12, "kv_heads": 12, "dim": 64, "causal": True, "ragged": True, "step": False},
        # Decoding two sequences over a long cache with shared key heads.
        {"name": "decode_f16_long", "kind": "attend", "form": "heads", "dtype": "f16", "batch": 2, "queries": 1,
         "keys": 65_536, "heads": 16, "kv_heads": 4, "dim": 128, "causal": True, "ragged": False, "step": False},
        # The MLP's activation in training on 8 sequences of 1024 tokens.
        {"name": "gelu_step_bf16_8k", "kind": "gelu", "dtype": "bf16", "rows": 8192, "features": 3072, "bias": True,
         "approximate": "none", "step": True},
        # The same at 16 decoded tokens in float16, nothing kept, with the tanh form of GELU.
        {"name": "gelu_f16_16", "kind": "gelu", "dtype": "f16", "rows": 16, "features": 3072, "bias": True,
         "approximate": "tanh", "step": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "attend", "attend", "attend", "gelu"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "norm":
        features = rng.choice([768, 3072, _log_int(rng, 16, 12_000)])
        return {"kind": kind, "dtype": dtype, "weight": rng.choice(["f32", dtype]),
                "rows": _log_int(rng, 1, min(16_384, 64_000_000 // features)), "features": features,
                "bias": rng.random() < 0.7, "residual": rng.random() < 0.5, "step": rng.random() < 0.6}
    if kind == "gelu":
        features = rng.choice([3072, _log_int(rng, 64, 8_192)])
        return {"kind": kind, "dtype": dtype, "rows": _log_int(rng, 1, min(16_384, 50_000_000 // features)),
                "features": features, "bias": rng.random() < 0.7, "approximate": rng.choice(["none", "tanh"]),
                "step": rng.random() < 0.6}
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    heads = kv_heads * (1 if kv_heads == 12 else rng.choice([1, 2, 3, 4]))
    dim = rng.choice([64, 64, 128, 32, 96, rng.randrange(8, 129)])
    what = rng.choice(["decode", "prefill", "step"])
    if what == "decode":  # one to four new tokens, caches of up to 2^17 tokens and 64 sequences
        keys = _log_int(rng, 16, 131_072)
        batch = _log_int(rng, 1, min(64, max(1, 60_000_000 // (keys * kv_heads * dim))))
        return {"kind": kind, "form": "heads", "dtype": dtype, "batch": batch, "queries": rng.choice([1, 1, 1, 2, 4]),
                "keys": keys, "heads": heads, "kv_heads": kv_heads, "dim": dim, "causal": True,
                "ragged": rng.random() < 0.6, "step": False}
    step = what == "step"
    # float32 products run at a sixteenth of the 16-bit ones' rate, a step has three and a half times
    # a forward's
    pairs = (1 << 28) // (heads * (4 if step else 1) * (8 if dtype == "f32" else 1))
    queries = _log_int(rng, 16, min(4096 if step else 8192, int(math.sqrt(pairs))))
    batch = _log_int(rng, 1, min(16, max(1, pairs // (queries * queries))))
    packed = rng.random() < 0.5
    keys = queries if packed else min(_log_int(rng, 16, 4096), max(16, pairs // (batch * queries)))
    return {"kind": kind, "form": "packed" if packed else "heads", "dtype": dtype, "batch": batch, "queries": queries,
            "keys": keys, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "causal": packed or (keys >= queries and rng.random() < 0.5),
            "ragged": not packed and rng.random() < 0.5, "step": step}


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _lengths(case):
    """Keys of each sequence: spread evenly from none to all of them where the batch is ragged."""
    b, keys = case["batch"], case["keys"]
    if not case["ragged"]:
        return [keys] * b
    least = 0 if case["queries"] > 1 else 1  # a sequence that decodes holds its own token at least
    return [max(least, round(keys * (i + 0.0 if b > 1 else 0.7) / max(1, b - 1))) for i in range(b)]


def prepare(case, seed):
    gen, dt = _generator(seed), DTYPES[case["dtype"]]

    def randn(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device=DEVICE) * std).to(dtype)

    state = {"case": case}
    if case["kind"] == "norm":
        rows, f = case["rows"], case["features"]
        wt = DTYPES[case["weight"]]
        # a residual stream: channels of different offset and size
        spread = torch.exp(0.5 * torch.randn(f, generator=gen, device=DEVICE))
        shift = 0.3 * torch.randn(f, generator=gen, device=DEVICE)
        state["x"] = (torch.randn(rows, f, generator=gen, device=DEVICE) * spread + shift).to(dt)
        state["weight"] = (1.0 + randn(f, std=0.1, dtype=torch.float32)).to(wt)
        state["bias"] = randn(f, std=0.1, dtype=wt) if case["bias"] else None
        state["residual"] = randn(rows, f) if case["residual"] else None
        if case["step"]:
            state["dy"] = randn(rows, f, std=0.05)
            state["dh"] = randn(rows, f, std=0.05) if case["residual"] else None
    elif case["kind"] == "gelu":
        rows, f = case["rows"], case["features"]
        spread = torch.exp(0.3 * torch.randn(f, generator=gen, device=DEVICE))
        state["x"] = (torch.randn(rows, f, generator=gen, device=DEVICE) * spread).to(dt)
        state["bias"] = randn(f, std=0.2) if case["bias"] else None
        if case["step"]:
            state["dy"] = randn(rows, f, std=0.05)
    else:
        b, tq, tk, h, hk, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
        if case["form"] == "packed":  # what the block's first linear leaves: queries, keys, values side by side
            state["qkv"] = randn(b, tq, (h + 2 * hk) * d)
            if case["step"]:
                state["do"] = randn(b, tq, h * d, std=0.05)
        else:  # a sequence's tokens lie one after the other, all heads of a token together
            state["q"] = randn(b, tq, h, d).transpose(1, 2)
            state["k"] = randn(b, tk, hk, d).transpose(1, 2)
            state["v"] = randn(b, tk, hk, d).transpose(1, 2)
            if case["step"]:
                state["do"] = randn(b, tq, h, d, std=0.05).transpose(1, 2)
            if case["ragged"]:
                lengths = _lengths(case)
                order = torch.randperm(b, generator=torch.Generator().manual_seed(seed)).tolist()
                state["lengths"] = torch.tensor([lengths[i] for i in order], dtype=torch.int32, device=DEVICE)
    if case["step"]:  # what a training program differentiates by
        for key in ("x", "weight", "bias", "residual", "qkv", "q", "k", "v"):
            if state.get(key) is not None:
                state[key] = state[key].detach().requires_grad_(True)
    return state


# ---------------------------------------------------------------- the framework's operators
def _run_own(state):
    import latent_weight_lab_amd as lwl

    case = state["case"]
    if case["kind"] == "norm":
        x, w, b, r = state["x"], state["weight"], state["bias"], state["residual"]
        out = lwl.layer_norm(x, w, b, eps=EPS, residual=r)
        outs = list(out) if r is not None else [out]
        if not case["step"]:
            return outs
        wanted = [x, w] + ([b] if b is not None else [])
        upstream = [state["dy"]] + ([state["dh"]] if r is not None else [])
        grads = torch.autograd.grad(outs, wanted, upstream)
        return [t.detach() for t in outs] + list(grads)
    if case["kind"] == "gelu":
        x, b = state["x"], state["bias"]
        if not case["step"]:
            return [lwl.gelu_checkpoint8(x, b, approximate=case["approximate"])]
        y, checkpoint = lwl.gelu_checkpoint8(x, b, approximate=case["approximate"], return_checkpoint=True)
        again = checkpoint.activation()
        grads = torch.autograd.grad(y, [x] + ([b] if b is not None else []), state["dy"])
        return [y.detach(), again] + list(grads)
    if case["form"] == "packed":
        inputs = [state["qkv"]]
        o = lwl.attention_packed(state["qkv"], case["heads"], case["kv_heads"], causal=case["causal"])
    else:
        inputs = [state["q"], state["k"], state["v"]]
        o = lwl.attention(*inputs, causal=case["causal"], key_lengths=state.get("lengths"))
    if not case["step"]:
        return [o]
    return [o.detach()] + list(torch.autograd.grad(o, inputs, state["do"]))


# ---------------------------------------------------------------- the same in elementary operations
def _gelu(z, approximate):
    """GELU and its derivative."""
    if approximate == "tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)
    phi = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))


def _checkpoint8(z):
    """What the 8-bit checkpoint of z stands for: groups of GROUP features under one scale each."""
    rows, f = z.shape
    pad = -f % GROUP
    zp = torch.cat([z, z.new_zeros(rows, pad)], dim=1) if pad else z
    zg = zp.view(rows, -1, GROUP)
    scale = zg.abs().amax(dim=-1, keepdim=True) * (1.0 / 127.0)
    codes = torch.round(zg * torch.where(scale > 0, scale.reciprocal(), torch.zeros_like(scale)))
    return (codes * scale).view(rows, f + pad)[:, :f]


def _split_heads(case, state):
    if case["form"] != "packed":
        return state["q"], state["k"], state["v"]
    b, t, h, hk, d = (case[k] for k in ("batch", "queries", "heads", "kv_heads", "dim"))
    q, k, v = state["qkv"].split([h * d, hk * d, hk * d], dim=-1)
    return (q.view(b, t, h, d).transpose(1, 2), k.view(b, t, hk, d).transpose(1, 2),
            v.view(b, t, hk, d).transpose(1, 2))


def _hidden(case, lengths, device):
    """True where a query may not see a key ([batch or 1, 1, queries, keys]), or None."""
    tq, tk = case["queries"], case["keys"]
    j = torch.arange(tk, device=device)
    if lengths is None:
        if not case["causal"]:
            return None
        i = torch.arange(tq, device=device).view(-1, 1) + (tk - tq)
        return (j > i).view(1, 1, tq, tk)
    n = lengths.view(-1, 1, 1, 1).long()
    hidden = (j >= n)
    if case["causal"]:  # the queries are the sequence's last tokens
        hidden = hidden | (j > torch.arange(tq, device=device).view(-1, 1) + (n - tq))
    return hidden.expand(-1, -1, tq, -1)


def _attend(case, q, k, v, do, hidden):
    """Output and, with ``do``, the gradients, in the type of q."""
    group = case["heads"] // case["kv_heads"]
    b, hk, tk, d = k.shape
    kx = k.repeat_interleave(group, dim=1) if group > 1 else k.contiguous()
    vx = v.repeat_interleave(group, dim=1) if group > 1 else v.contiguous()
    scale = 1.0 / math.sqrt(d)
    s = torch.matmul(q.contiguous(), kx.transpose(2, 3).contiguous()) * scale
    if hidden is not None:
        s = s.masked_fill(hidden, float("-inf"))
    top = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.matmul(p, vx)
    if do is None:
        return o, ()
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    dp = torch.matmul(do, vx.transpose(2, 3).contiguous())
    ds = p * (dp - (do * o).sum(dim=-1, keepdim=True)) * scale
    dq = torch.matmul(ds, kx)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q.contiguous())
    if group > 1:
        dk, dv = (t.view(b, hk, group, tk, d).sum(dim=2) for t in (dk, dv))
    return o, (dq, dk, dv)


def _norm(x, w, b, r, dy, dh, dt):
    """Outputs and gradients of the norm in the type of x; ``dt``: the type the sum is kept in."""
    h = x if r is None else (x + r).to(dt).to(x.dtype)
    mean = h.mean(dim=-1, keepdim=True)
    c = h - mean
    rstd = torch.rsqrt((c * c).mean(dim=-1, keepdim=True) + EPS)
    n = c * rstd
    y = n * w if b is None else n * w + b
    outs = [y] if r is None else [y, h]
    if dy is None:
        return outs
    a = dy * w
    dx = rstd * (a - a.mean(dim=-1, keepdim=True) - n * (a * n).mean(dim=-1, keepdim=True))
    if dh is not None:
        dx = dx + dh
    return outs + [dx, (dy * n).sum(dim=0)] + ([dy.sum(dim=0)] if b is not None else [])


def _compute(state, ft, round_sum):
    """An operator in elementary operations in the type ``ft``, outputs in it too."""
    case, dt = state["case"], DTYPES[state["case"]["dtype"]]

    def wide(key):
        return state[key].detach().to(ft) if state.get(key) is not None else None

    if case["kind"] == "norm":
        return _norm(wide("x"), wide("weight"), wide("bias"), wide("residual"), wide("dy"), wide("dh"),
                     dt if round_sum else ft)
    if case["kind"] == "gelu":
        z = wide("x")
        if case["bias"]:
            z = z + wide("bias")
        y = _gelu(z, case["approximate"])[0]
        if not case["step"]:
            return [y]
        again, slope = _gelu(_checkpoint8(z), case["approximate"])
        dx = wide("dy") * slope
        return [y, again, dx] + ([dx.sum(dim=0)] if case["bias"] else [])
    b, tq, d = case["batch"], case["queries"], case["dim"]
    q, k, v = (t.detach().to(ft) for t in _split_heads(case, state))
    do = wide("do")
    if do is not None and case["form"] == "packed":
        do = do.view(b, tq, case["heads"], d).transpose(1, 2)
    if do is not None:
        do = do.contiguous()
    o, grads = _attend(case, q, k, v, do, _hidden(case, state.get("lengths"), q.device))
    if case["form"] == "packed":
        o = o.transpose(1, 2).reshape(b, tq, -1)
        if grads:
            grads = [torch.cat([g.transpose(1, 2).reshape(b, tq, -1) for g in grads], dim=-1)]
    return [o] + list(grads)


def _types(case):
    """The outputs' types, in order."""
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "norm" and case["step"]:
        wt = DTYPES[case["weight"]]
        return [dt] * (3 if case["residual"] else 2) + [wt] * (2 if case["bias"] else 1)
    return [dt] * 4


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return [t.to(dt) for t, dt in zip(_compute(state, torch.float32, True), _types(state["case"]))]


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return _exact_norm(state) if case["kind"] == "norm" else (
            _exact_gelu(state) if case["kind"] == "gelu" else _exact_attend(state))


def _doubles(state, *keys):
    return [None if state.get(k) is None else state[k].detach().double() for k in keys]


def _exact_norm(state):
    case = state["case"]
    x, w, b, r, dy, dh = _doubles(state, "x", "weight", "bias", "residual", "dy", "dh")
    # the sum of the streams is an output of the input's type: what is normed is what is stored
    h = x if r is None else (state["x"].detach().float() + state["residual"].detach().float()).to(state["x"].dtype).double()
    f = h.shape[1]
    mean = h.sum(1, keepdim=True) / f
    var = ((h - mean) ** 2).sum(1, keepdim=True) / f
    sd = torch.sqrt(var + EPS)
    n = (h - mean) / sd
    out = [n * w + (0.0 if b is None else b)] + ([] if r is None else [x + r])
    if not case["step"]:
        return out
    g = dy * w
    inner = g.sum(1, keepdim=True) + n * (g * n).sum(1, keepdim=True)
    dx = (f * g - inner) / (f * sd) + (0.0 if dh is None else dh)
    return out + [dx, torch.einsum("rf,rf->f", dy, n)] + ([] if b is None else [dy.sum(0)])


def _exact_gelu(state):
    case = state["case"]
    x, b, dy = _doubles(state, "x", "bias", "dy")
    z = x if b is None else x + b

    def value(u):
        if case["approximate"] == "tanh":  # u * sigmoid(2 t) = u (1 + tanh t) / 2
            return u * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (u + 0.044715 * u ** 3))
        return 0.5 * u * torch.erfc(-u / math.sqrt(2.0))

    def slope(u):
        if case["approximate"] == "tanh":
            k = 2 * math.sqrt(2 / math.pi)
            s = torch.sigmoid(k * (u + 0.044715 * u ** 3))
            return s + u * s * (1 - s) * k * (1 + 0.134145 * u * u)
        return 0.5 * torch.erfc(-u / math.sqrt(2.0)) + u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi)

    if not case["step"]:
        return [value(z)]
    kept = torch.empty_like(z)
    for f0 in range(0, z.shape[1], GROUP):
        part = z[:, f0:f0 + GROUP]
        top = part.abs().max(dim=1, keepdim=True).values
        unit = torch.where(top > 0, top, torch.ones_like(top)) / 127
        kept[:, f0:f0 + GROUP] = torch.round(part / unit) * unit
    dx = dy * slope(kept)
    return [value(z), value(kept), dx] + ([] if b is None else [dx.sum(0)])


def _exact_attend(state):
    case = state["case"]
    b, tq, tk, h, hk, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    if case["form"] == "packed":
        x = state["qkv"].detach().double().view(b, tq, h + 2 * hk, d)
        q, k, v = x[:, :, :h], x[:, :, h:h + hk], x[:, :, h + hk:]
    else:
        q, k, v = (state[n].detach().double().transpose(1, 2) for n in ("q", "k", "v"))  # [b, t, heads, d]
    do = state["do"].detach().double() if case["step"] else None
    if do is not None:
        do = do.view(b, tq, h, d) if case["form"] == "packed" else do.transpose(1, 2)
    lengths = state["lengths"].tolist() if case["ragged"] else [tk] * b
    o = torch.zeros(b, tq, h, d, dtype=torch.float64, device=q.device)
    dq, dk, dv = (torch.zeros_like(t) for t in (q, k, v)) if case["step"] else (None, None, None)
    for bi in range(b):
        n = lengths[bi]
        if n == 0:
            continue
        for hi in range(h):
            ki = hi * hk // h
            kb, vb, qb = k[bi, :n, ki], v[bi, :n, ki], q[bi, :, hi]
            s = (qb @ kb.t()) / math.sqrt(d)
            seen = torch.ones(tq, n, dtype=torch.bool, device=q.device)
            if case["causal"]:
                seen = seen.tril(n - tq)
            s = torch.where(seen, s, -math.inf)
            log_sum = torch.logsumexp(s, dim=1, keepdim=True)
            p = torch.where(seen, torch.exp(s - torch.where(log_sum > -math.inf, log_sum, 0.0)), 0.0)
            o[bi, :, hi] = p @ vb
            if do is not None:
                g = do[bi, :, hi]
                dv[bi, :n, ki] += p.t() @ g
                ds = p * (g @ vb.t() - (g * o[bi, :, hi]).sum(1, keepdim=True)) / math.sqrt(d)
                dq[bi, :, hi] = ds @ kb
                dk[bi, :n, ki] += ds.t() @ qb
    if case["form"] == "packed":
        grads = [] if do is None else [torch.cat([t.reshape(b, tq, -1) for t in (dq, dk, dv)], dim=-1)]
        return [o.reshape(b, tq, h * d)] + grads
    return [t.transpose(1, 2) for t in ([o] if do is None else [o, dq, dk, dv])]


# ---------------------------------------------------------------- what the mathematics needs
def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["kind"] == "norm":
        n, ws = case["rows"] * case["features"], torch.finfo(DTYPES[case["weight"]]).bits // 8
        streams = 2 + (2 if case["residual"] else 0)  # x, y (residual and its sum)
        vectors = 1 + case["bias"]
        if case["step"]:  # dy, dx, with a residual the gradient of its sum too; the vectors' gradients
            streams += 2 + case["residual"]
            vectors *= 2
        return {"bytes": n * streams * size + vectors * case["features"] * ws, "flops": n * (20 if case["step"] else 8)}
    if case["kind"] == "gelu":
        n = case["rows"] * case["features"]
        vectors = case["features"] * size * case["bias"]
        if not case["step"]:
            return {"bytes": n * 2 * size + vectors, "flops": n * 12}
        # x, y, the activation again, dy, dx; the checkpoint written and read
        kept = n + case["rows"] * -(-case["features"] // GROUP) * 4
        return {"bytes": n * 5 * size + 2 * kept + 2 * vectors, "flops": n * 50}
    b, tq, h, hk, d = (case[k] for k in ("batch", "queries", "heads", "kv_heads", "dim"))
    lengths = _lengths(case)
    pairs = 0
    for n in lengths:
        if case["causal"]:  # query i sees n - tq + i + 1 keys, none where that is negative
            least, most = n - tq + 1, n
            rows = tq if least > 0 else max(0, most)
            pairs += rows * (max(least, 1) + most) // 2
        else:
            pairs += tq * n
    rows_q, rows_k = b * tq * h * d, sum(lengths) * hk * d
    if not case["step"]:
        return {"bytes": size * 2 * (rows_q + rows_k), "flops": 4 * pairs * h * d}
    # the step: q, o, do, dq and k, v, dk, dv; two products forward, five backward; gradients of keys
    # past a sequence's end are written as zeros
    return {"bytes": size * (4 * rows_q + 2 * rows_k + 2 * b * case["keys"] * hk * d), "flops": 14 * pairs * h * d}
