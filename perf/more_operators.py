"""Attention over long caches and drafted tokens, and the probabilities of tokens, as workloads for measurement.

Three operators, each through the package's public entry points:

``window``  attention within a sliding window whose first tokens stay visible: a prompt's forward, training
            steps, and new tokens over a cache
``tree``    attention of a tree of drafted tokens over a cache: every node sees what came before the tree, its
            ancestors and itself
``tokens``  log probabilities of given tokens with the entropy and the most probable alternatives: forward for
            decoding and for verifying drafts, forward and backward for training

``own`` chooses between the framework's operators and the same mathematics in elementary torch
operations in float32.  ``exact()`` restates each of them in float64.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda"
MOST_SCORES = 1 << 30  # scores that the plain forms hold at a time


def _window(name, form, dtype, batch, queries, keys, heads, kv_heads, dim, window, sinks, ragged, step):
    return {"name": name, "kind": "window", "form": form, "dtype": dtype, "batch": batch, "queries": queries, "keys": keys,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks, "ragged": ragged,
            "step": step}


def _tree(name, dtype, batch, nodes, keys, heads, kv_heads, dim, shape, ragged):
    return {"name": name, "kind": "tree", "dtype": dtype, "batch": batch, "queries": nodes, "keys": keys, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "shape": shape, "ragged": ragged, "step": False}


def _tokens(name, dtype, rows, vocab, pitch, each, entropy, top, step):
    return {"name": name, "kind": "tokens", "dtype": dtype, "rows": rows, "vocab": vocab, "pitch": pitch, "each": each,
            "entropy": entropy, "top": top, "step": step}


def listed():
    return [
        # A training step of GPT-2 small's attention on 8 sequences of 1024 tokens, local to 256 of them.
        _window("window_step_bf16_8x1024", "packed", "bf16", 8, 1024, 1024, 12, 12, 64, 256, 4, False, True),
        # The same on short sequences in float32 (a check of numerics, a small model).
        _window("window_step_f32_4x512", "packed", "f32", 4, 512, 512, 12, 12, 64, 128, 0, False, True),
        # A training step over padded sequences, one of them empty, after cached tokens, with key heads shared by
        # three query heads, a head size that fills no tile and a window of odd length.
        _window("window_step_f16_ragged", "heads", "f16", 6, 515, 1531, 12, 4, 80, 333, 7, True, True),
        # One long prompt, key heads shared by four query heads: the most pairs of all.
        _window("window_prefill_bf16_1x16384", "heads", "bf16", 1, 16_384, 16_384, 16, 4, 128, 4096, 4, False, False),
        # Decoding 64 sequences of different lengths over caches of up to 8192 tokens, one token each.
        _window("window_decode_bf16_64", "heads", "bf16", 64, 1, 8192, 12, 12, 64, 1024, 4, True, False),
        # 16 drafted tokens of one sequence over GPT-2 small's cache.
        _tree("tree_bf16_1x16", "bf16", 1, 16, 1024, 12, 12, 64, "wide", False),
        # 16 sequences of different lengths with 32 drafted tokens each, key heads shared by four query heads.
        _tree("tree_bf16_16x32", "bf16", 16, 32, 8192, 16, 4, 128, "wide", True),
        # 61 drafted tokens over one long cache, key heads shared by eight query heads.
        _tree("tree_f16_long", "f16", 1, 61, 65_536, 16, 2, 128, "deep", False),
        # Choosing the next token of 16 sequences: its probability, the entropy, five alternatives.
        _tokens("tokens_bf16_16", "bf16", 16, 50_304, 50_304, 1, True, 5, False),
        # Verifying 32 drafted tokens of 16 sequences: up to four children of every node, and what the model would say.
        _tokens("tokens_verify_bf16_512", "bf16", 512, 50_304, 50_304, 4, False, 1, False),
        # The training loss of 8 sequences of 1024 tokens over GPT-2's vocabulary, rows padded to 50304: the most bytes.
        _tokens("tokens_step_bf16_8k", "bf16", 8192, 50_257, 50_304, 1, False, 0, True),
        # A policy's step in float32: log probabilities and entropies, over another vocabulary of odd size.
        _tokens("tokens_step_f32_entropy", "f32", 1021, 32_003, 32_003, 1, True, 0, True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    case = _draw(rng)
    del case["name"]
    return case


def _draw(rng):
    kind = rng.choice(["window", "window", "tree", "tree", "tokens", "tokens"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "tokens":
        vocab = rng.choice([50_257, 50_304, _log_int(rng, 128, 200_000)])
        step = rng.random() < 0.5
        top = 0 if step else rng.choice([0, 1, 5, 20, rng.randrange(1, 33)])
        most = 400_000_000 // (2 if dtype == "f32" else 1) // (8 if top else 1)
        return _tokens("", dtype, _log_int(rng, 1, min(8192, most // vocab)), vocab,
                       vocab + rng.choice([0, 0, rng.randrange(1, 64)]), rng.choice([1, 1, 1, rng.randrange(2, 9)]),
                       rng.random() < 0.5, top, step)
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    heads = kv_heads * (1 if kv_heads == 12 else rng.choice([1, 2, 3, 4]))
    dim = rng.choice([64, 64, 128, 32, 96, rng.randrange(8, 129)])
    if kind == "tree":
        keys = _log_int(rng, 160, 131_072)
        batch = _log_int(rng, 1, min(64, max(1, 60_000_000 // (keys * kv_heads * dim))))
        nodes = rng.choice([16, 32, 64, _log_int(rng, 1, 128)])
        return _tree("", dtype, batch, nodes, keys, heads, kv_heads, dim, rng.choice(["wide", "deep", "chain"]),
                     rng.random() < 0.6)
    window, sinks = _log_int(rng, 16, 4096), rng.choice([0, 1, 4, rng.randrange(0, 100)])
    what = rng.choice(["decode", "prefill", "step"])
    if what == "decode":  # one to four new tokens, caches of up to 2^17 tokens and 64 sequences
        keys = _log_int(rng, 16, 131_072)
        batch = _log_int(rng, 1, min(64, max(1, 60_000_000 // (keys * kv_heads * dim))))
        return _window("", "heads", dtype, batch, rng.choice([1, 1, 1, 2, 4]), keys, heads, kv_heads, dim, window, sinks,
                       rng.random() < 0.6, False)
    step = what == "step"
    # float32 products run at a sixteenth of the 16-bit ones' rate, a step has three and a half times
    # a forward's; the plain forms make every pair
    pairs = (1 << 28) // (heads * (4 if step else 1) * (8 if dtype == "f32" else 1))
    queries = _log_int(rng, 16, min(4096 if step else 8192, int(math.sqrt(pairs))))
    batch = _log_int(rng, 1, min(16, max(1, pairs // (queries * queries))))
    packed = rng.random() < 0.5
    keys = queries if packed else max(queries, min(_log_int(rng, 16, 4096), pairs // (batch * queries)))
    return _window("", "packed" if packed else "heads", dtype, batch, queries, keys, heads, kv_heads, dim, window, sinks,
                   not packed and rng.random() < 0.5, step)


def _lengths(case):
    """Keys of each sequence: spread evenly from none to all of them where the batch is ragged."""
    b, keys = case["batch"], case["keys"]
    if not case["ragged"]:
        return [keys] * b
    # a sequence that decodes holds its own new tokens at least
    least = case["queries"] if case["kind"] == "tree" or case["queries"] <= 4 else 0
    least = min(least, keys)
    return [max(least, round(keys * (i + 0.0 if b > 1 else 0.7) / max(1, b - 1))) for i in range(b)]


def _parents(case, seed):
    """A tree for each sequence: nodes that follow one of the few before them, with few or many at a depth."""
    n, b = case["queries"], case["batch"]
    rng = np.random.default_rng(seed)
    back = {"chain": np.ones((b, n), dtype=np.int64), "deep": rng.integers(1, 5, (b, n)),
            "wide": np.arange(n)[None] - np.arange(n)[None] // rng.integers(2, 5, (b, 1))}[case["shape"]]
    parents = np.arange(n)[None] - back
    parents[:, 0] = -1
    return np.clip(parents, -1, np.maximum(np.arange(n) - 1, -1)).astype(np.int32)


def prepare(case, seed):
    gen, dt = torch.Generator(device=DEVICE).manual_seed(seed), DTYPES[case["dtype"]]

    def randn(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device=DEVICE) * std).to(dtype)

    state = {"case": case}
    if case["kind"] == "tokens":
        rows, vocab, each = case["rows"], case["vocab"], case["each"]
        shape = (rows,) if each == 1 else (rows, each)
        tokens = torch.randint(vocab, shape, generator=gen, device=DEVICE)
        logits = torch.empty(rows, case["pitch"], dtype=dt, device=DEVICE)
        wide = torch.randn(rows, vocab, generator=gen, device=DEVICE) * 2.0
        # about half of the rows are fairly sure of what is asked about, the others know nothing of it
        sure = torch.rand(rows, 1, generator=gen, device=DEVICE)
        first = tokens.view(rows, each)[:, :1]
        wide.scatter_add_(1, first, 16.0 * (sure - 0.5).clamp_min(0.0) * 2.0)
        logits[:, :vocab] = wide.to(dt)
        logits[:, vocab:] = float("nan")
        del wide
        # padding: the ends of sequences, nodes without that many children
        tokens = tokens.masked_fill(torch.rand(shape, generator=gen, device=DEVICE) < 0.1, -1)
        state["logits"], state["tokens"] = logits[:, :vocab], tokens
        if case["step"]:
            state["logits"] = logits[:, :vocab].detach().requires_grad_(True)
            state["g"] = randn(*shape, std=1.0 / rows, dtype=torch.float32)
            state["gh"] = randn(rows, std=0.1 / rows, dtype=torch.float32) if case["entropy"] else None
        return state
    b, tq, tk, h, hk, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    if case.get("form") == "packed":  # what the block's first linear leaves: queries, keys, values side by side
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
    if case["kind"] == "tree":
        state["parents"] = torch.from_numpy(_parents(case, seed)).to(DEVICE)
    if case["step"]:  # what a training program differentiates by
        for key in ("qkv", "q", "k", "v"):
            if key in state:
                state[key] = state[key].detach().requires_grad_(True)
    return state


# ---------------------------------------------------------------- the framework's operators
def _run_own(state):
    import latent_weight_lab_amd as lwl

    case = state["case"]
    if case["kind"] == "tokens":
        out = lwl.token_log_probs(state["logits"], state["tokens"], entropy=case["entropy"], top=case["top"])
        out = list(out) if isinstance(out, tuple) else [out]
        if not case["step"]:
            return out
        upstream = [state["g"]] + ([state["gh"]] if case["entropy"] else [])
        return [t.detach() for t in out] + list(torch.autograd.grad(out, [state["logits"]], upstream))
    if case["kind"] == "tree":
        return [lwl.attention_tree(state["q"], state["k"], state["v"], state["parents"], key_lengths=state.get("lengths"))]
    if case["form"] == "packed":
        inputs = [state["qkv"]]
        o = lwl.attention_packed(state["qkv"], case["heads"], case["kv_heads"], window=case["window"], sinks=case["sinks"])
    else:
        inputs = [state["q"], state["k"], state["v"]]
        o = lwl.attention(*inputs, causal=True, key_lengths=state.get("lengths"), window=case["window"],
                          sinks=case["sinks"])
    if not case["step"]:
        return [o]
    return [o.detach()] + list(torch.autograd.grad(o, inputs, state["do"]))


# ---------------------------------------------------------------- the same in elementary operations
def _split_heads(case, state):
    if case.get("form") != "packed":
        return state["q"], state["k"], state["v"]
    b, t, h, hk, d = (case[k] for k in ("batch", "queries", "heads", "kv_heads", "dim"))
    q, k, v = state["qkv"].split([h * d, hk * d, hk * d], dim=-1)
    return (q.view(b, t, h, d).transpose(1, 2), k.view(b, t, hk, d).transpose(1, 2),
            v.view(b, t, hk, d).transpose(1, 2))


def _hidden(case, state):
    """True where a query may not see a key: [batch or 1, 1, queries, keys]."""
    tq, tk = case["queries"], case["keys"]
    j = torch.arange(tk, device=DEVICE).view(1, 1, 1, tk)
    n = state["lengths"].long() if state.get("lengths") is not None else torch.full((1,), tk, device=DEVICE)
    n = n.view(-1, 1, 1, 1)
    first = n - tq  # position of the first query
    if case["kind"] == "window":
        p = first + torch.arange(tq, device=DEVICE).view(1, 1, tq, 1)
        return (j >= n) | (j > p) | ((j <= p - case["window"]) & (j >= case["sinks"]))
    # a node's row holds its parent's row and itself
    parents = state["parents"].long()
    b = parents.shape[0]
    line = torch.eye(tq, dtype=torch.bool, device=DEVICE).expand(b, tq, tq).clone()
    up = parents
    for _ in range(max(1, tq - 1).bit_length()):  # everything 1, 2, 4, .. steps up
        have = up >= 0
        above = up.clamp_min(0)
        line = line | (torch.gather(line, 1, above.unsqueeze(-1).expand(-1, -1, tq)) & have.unsqueeze(-1))
        up = torch.where(have, torch.gather(up, 1, above), up)
    node = (j - first).expand(b, 1, tq, tk)
    in_tree = torch.gather(line.unsqueeze(1), 3, node.clamp(0, tq - 1))
    return torch.where(node < 0, False, ~in_tree) | (node >= tq)


def _attend(case, q, k, v, do, hidden):
    """Output and, with ``do``, the gradients."""
    group = case["heads"] // case["kv_heads"]
    b, hk, tk, d = k.shape
    kx = k.repeat_interleave(group, dim=1) if group > 1 else k.contiguous()
    vx = v.repeat_interleave(group, dim=1) if group > 1 else v.contiguous()
    scale = 1.0 / math.sqrt(d)
    s = torch.matmul(q.contiguous(), kx.transpose(2, 3).contiguous()) * scale
    s = s.masked_fill(hidden, float("-inf"))
    top = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.matmul(p, vx)
    if do is None:
        return [o]
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    dp = torch.matmul(do, vx.transpose(2, 3).contiguous())
    ds = p * (dp - (do * o).sum(dim=-1, keepdim=True)) * scale
    dq = torch.matmul(ds, kx)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q.contiguous())
    if group > 1:
        dk, dv = (t.view(b, hk, group, tk, d).sum(dim=2) for t in (dk, dv))
    return [o, dq, dk, dv]


def _attend_parts(case, q, k, v, do, hidden):
    """The same a few sequences and key heads at a time, so that the scores fit."""
    b, h, tq, _ = q.shape
    hk, tk, group = k.shape[1], k.shape[2], case["heads"] // case["kv_heads"]
    if b * h * tq * tk <= MOST_SCORES:
        return _attend(case, q, k, v, do, hidden)
    parts = []
    for bi in range(b):
        for ki in range(hk):
            heads, one = slice(ki * group, (ki + 1) * group), slice(bi, bi + 1)
            parts.append(_attend(case, q[one, heads], k[one, ki:ki + 1], v[one, ki:ki + 1],
                                 None if do is None else do[one, heads], hidden if hidden.shape[0] == 1 else hidden[one]))
    whole = [torch.cat([p[i] for p in parts], dim=1) for i in range(len(parts[0]))]
    return [w.view(b, n, *w.shape[2:]) for w, n in zip(whole, (h, h, hk, hk))]


def _judge(case, logits, tokens, g, gh):
    """Log probabilities, entropy, the top ones; with ``g`` the logits' gradient."""
    m = logits.amax(dim=-1, keepdim=True)
    z = logits - m
    e = torch.exp(z)
    total = e.sum(dim=-1, keepdim=True)
    log_total = torch.log(total)
    each = tokens.view(tokens.shape[0], -1)
    asked = each >= 0
    out = [torch.where(asked, torch.gather(z, 1, each.clamp_min(0)) - log_total, 0.0).view(tokens.shape)]
    entropy = None
    if case["entropy"]:
        entropy = log_total - (e * z).sum(dim=-1, keepdim=True) / total
        out.append(entropy.squeeze(-1))
    if case["top"]:
        rest, values, where = z.clone(), [], []
        for _ in range(case["top"]):  # the largest that is left, the first of equal ones
            value, index = rest.max(dim=-1)
            values.append(value - log_total.squeeze(-1))
            where.append(index)
            rest.scatter_(1, index.unsqueeze(-1), float("-inf"))
        out += [torch.stack(values, -1), torch.stack(where, -1)]
    if g is None:
        return out
    g = torch.where(asked, g.view(each.shape), 0.0)
    p = e / total
    dz = -p * g.sum(dim=-1, keepdim=True)
    if gh is not None:
        dz = dz - gh.unsqueeze(-1) * p * (z - log_total + entropy)
    return out + [dz.scatter_add_(1, each.clamp_min(0), g)]


def run(state):
    if own:
        return _run_own(state)
    case, dt = state["case"], DTYPES[state["case"]["dtype"]]
    with torch.no_grad():
        if case["kind"] == "tokens":
            out = _judge(case, state["logits"].detach().float(), state["tokens"], state.get("g"), state.get("gh"))
            return out[:-1] + [out[-1].to(dt)] if case["step"] else out
        b, tq, d = case["batch"], case["queries"], case["dim"]
        q, k, v = (t.detach().float() for t in _split_heads(case, state))
        do = state["do"].float() if case["step"] else None
        if do is not None and case["form"] == "packed":
            do = do.view(b, tq, case["heads"], d).transpose(1, 2)
        out = _attend_parts(case, q, k, v, None if do is None else do.contiguous(), _hidden(case, state))
        if case.get("form") == "packed":
            out = [t.transpose(1, 2).reshape(b, tq, -1) for t in out]
            out = out[:1] + ([torch.cat(out[1:], dim=-1)] if case["step"] else [])
        return [t.to(dt) for t in out]


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return _exact_tokens(state) if case["kind"] == "tokens" else _exact_attend(state)


def _exact_tokens(state):
    case = state["case"]
    x, tokens = state["logits"].detach().double(), state["tokens"]
    rows = x.shape[0]
    log_p = x - torch.logsumexp(x, 1, keepdim=True)
    each = tokens.reshape(rows, -1)
    lp = torch.zeros(each.shape, dtype=torch.float64, device=x.device)
    r, c = torch.nonzero(each >= 0, as_tuple=True)
    lp[r, c] = log_p[r, each[r, c]]
    out = [lp.view(tokens.shape)]
    p = torch.exp(log_p)
    entropy = -torch.where(p > 0, p * log_p, 0.0).sum(1)
    if case["entropy"]:
        out.append(entropy)
    if case["top"]:
        values, order = torch.sort(x, dim=1, descending=True, stable=True)
        out += [torch.gather(log_p, 1, order[:, :case["top"]]), order[:, :case["top"]].clone()]
        del values, order
    if not case["step"]:
        return out
    g = state["g"].double().view(rows, -1) * (each >= 0)
    dz = -p * g.sum(1, keepdim=True)
    dz.index_put_((r, each[r, c]), g[r, c], accumulate=True)
    if case["entropy"]:
        dz -= state["gh"].double().unsqueeze(1) * p * (log_p + entropy.unsqueeze(1))
    return out + [dz]


def _exact_attend(state):
    case = state["case"]
    b, tq, tk, h, hk, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    if case.get("form") == "packed":
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
        seen = np.zeros((tq, n), dtype=bool)
        if case["kind"] == "tree":
            parents = state["parents"][bi].tolist()
            for i in range(tq):
                seen[i, :max(0, n - tq)] = True
                at = i
                while at >= 0:
                    if n - tq + at >= 0:
                        seen[i, n - tq + at] = True
                    at = parents[at]
        else:
            for i in range(tq):
                p = n - tq + i
                if p >= 0:
                    seen[i, :min(case["sinks"], p + 1)] = True
                    seen[i, max(0, p - case["window"] + 1):p + 1] = True
        seen = torch.from_numpy(seen).to(q.device)
        for hi in range(h):
            ki = hi * hk // h
            kb, vb, qb = k[bi, :n, ki], v[bi, :n, ki], q[bi, :, hi]
            s = (qb @ kb.t()) / math.sqrt(d)
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
    if case.get("form") == "packed":
        grads = [] if do is None else [torch.cat([t.reshape(b, tq, -1) for t in (dq, dk, dv)], dim=-1)]
        return [o.reshape(b, tq, h * d)] + grads
    return [t.transpose(1, 2) for t in ([o] if do is None else [o, dq, dk, dv])]


# ---------------------------------------------------------------- what the mathematics needs
def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["kind"] == "tokens":
        n, rows = case["rows"] * case["vocab"], case["rows"]
        small = rows * (case["each"] * 12 + 4 * case["entropy"] + 12 * case["top"])
        if not case["step"]:
            return {"bytes": n * size + small, "flops": n * (4 + 2 * case["entropy"])}
        # the logits once and their gradient once (rows of any vocabulary do not stay on chip between the passes of
        # a step, but nothing in the mathematics reads them twice)
        return {"bytes": 2 * n * size + small + 4 * rows * (case["each"] + case["entropy"]),
                "flops": n * (8 + 6 * case["entropy"])}
    b, tq, h, hk, d = (case[k] for k in ("batch", "queries", "heads", "kv_heads", "dim"))
    lengths = _lengths(case)
    pairs, cached = 0, 0  # pairs of a query and a key it sees; keys that some query sees
    depths = None
    if case["kind"] == "tree":
        parents = _parents(case, 0)
        depths = np.zeros(parents.shape, dtype=np.int64)
        for i in range(tq):
            above = parents[:, i]
            depths[:, i] = np.where(above >= 0, np.take_along_axis(depths, np.maximum(above, 0)[:, None], 1)[:, 0], 0) + 1
    for bi, n in enumerate(lengths):
        p = np.arange(tq, dtype=np.int64) + n - tq
        if depths is not None:
            pairs += int(depths[bi].sum()) + tq * max(0, n - tq)
            cached += n
        else:
            p = p[p >= 0]
            if len(p):
                first = np.maximum(0, p - case["window"] + 1)
                pairs += int((p + 1 - first + np.minimum(first, case["sinks"])).sum())
                cached += int(n - first[0] + min(first[0], case["sinks"]))
    rows_q, rows_k = b * tq * h * d, cached * hk * d
    if not case["step"]:
        return {"bytes": size * 2 * (rows_q + rows_k), "flops": 4 * pairs * h * d}
    # the step: q, o, do, dq and k, v, dk, dv; two products forward, five backward; gradients of keys
    # that no query sees are written as zeros
    return {"bytes": size * (4 * rows_q + 2 * rows_k + 2 * b * case["keys"] * hk * d), "flops": 14 * pairs * h * d}
