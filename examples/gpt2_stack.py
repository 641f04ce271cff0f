"""A GPT-2 shaped stack of generated linears with the operators between them: a training step and decoding.

    python examples/gpt2_stack.py                      # 12 layers of 768, bfloat16: a training step, then decoding
    python examples/gpt2_stack.py --layers 2 --batch 2
    python examples/gpt2_stack.py --window 256 --sinks 4   # attention local to 256 tokens and the first 4

The four linears of a block are ``BlockFHTLinear``s (reference ``examples/nanogpt/model.py``), used through
the weight cache: weights are generated once a step, and their gradients projected onto the latents
once.  Between them, each in one pass over its data: the residual addition with the layer norm, attention
straight from one linear's output to the next one's input, and the GELU that keeps 8 bits of its input.  The
loss is the log probabilities of the next tokens, read from the logits as they are.  Decoding takes one token at a
time, or a tree of drafts, judged together in one pass over the cache.  Random weights and tokens.
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch
import torch.nn.functional as F
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import latent_weight_lab_amd as lwl  # noqa: E402


class Block(nn.Module):
    def __init__(self, width: int, heads: int, latent_ratio: float, seed: int) -> None:
        super().__init__()
        self.heads = heads
        self.norm1, self.norm2 = lwl.LayerNorm(width), lwl.LayerNorm(width)

        def linear(n_in, n_out, k):
            # rows of unit variance become rows of variance about 1/3, a usual initialization's
            return lwl.BlockFHTLinear(n_in, n_out, latent_ratio=latent_ratio, seed=4 * seed + k, latent_init_std=1.0,
                                      weight_scale=(3 * n_in) ** -0.5)

        self.qkv, self.proj = linear(width, 3 * width, 0), linear(width, width, 1)
        self.up, self.down = linear(width, 4 * width, 2), linear(4 * width, width, 3)
        self.up_bias = nn.Parameter(torch.zeros(4 * width))

    def forward(self, delta, stream, attend):
        """``stream`` is the residual stream without ``delta``, what the block before adds to it; returns both
        for the next block.  ``attend(qkv)`` is the attention of this block."""
        n, stream = self.norm1(delta, stream)
        n, stream = self.norm2(self.proj(attend(self.qkv(n))), stream)
        return lwl.gelu_linear_checkpoint8(self.up(n), self.down, self.up_bias, approximate="tanh"), stream


class Cache:
    """Keys and values of one block, ``[batch, heads, capacity, head size]``."""

    def __init__(self, batch, heads, capacity, head_size, like, local=None):
        self.k, self.v = (like.new_empty(batch, heads, capacity, head_size) for _ in range(2))
        self.local = local or {}  # attention's window and sinks

    def split(self, qkv):
        batch, tokens, _ = qkv.shape
        return qkv.view(batch, tokens, 3, self.k.shape[1], -1).permute(2, 0, 3, 1, 4)

    def prompt(self, qkv, lengths):
        """Attention of prompts padded at their ends, which become the cache's first tokens."""
        _, k, v = self.split(qkv)
        self.k[:, :, :qkv.shape[1]], self.v[:, :, :qkv.shape[1]] = k, v
        return lwl.attention_packed(qkv, self.k.shape[1], key_lengths=lengths, causal_offset=0, **self.local)

    def token(self, qkv, lengths):
        """Attention of one new token for each sequence over what the cache holds of it and itself."""
        q, k, v = self.split(qkv)
        rows = torch.arange(len(lengths), device=lengths.device)
        self.k[rows, :, lengths], self.v[rows, :, lengths] = k[:, :, 0], v[:, :, 0]
        out = lwl.attention(q, self.k, self.v, causal=True, key_lengths=lengths + 1, **self.local)
        return out.transpose(1, 2).reshape(qkv.shape[0], 1, -1)

    def at(self, places):
        """Indexes of ``places`` (``[batch, tokens]``), the heads' axis last but one."""
        return torch.arange(len(places), device=places.device)[:, None], slice(None), places

    def drafts(self, qkv, lengths, parents):
        """Attention of a tree of drafted tokens, whose keys and values follow what the cache holds."""
        q, k, v = self.split(qkv)
        nodes = qkv.shape[1]
        at = self.at(lengths[:, None] + torch.arange(nodes, device=lengths.device))
        self.k[at], self.v[at] = k.transpose(1, 2), v.transpose(1, 2)
        out = lwl.attention_tree(q, self.k, self.v, parents, key_lengths=lengths + nodes)
        return out.transpose(1, 2).reshape(*qkv.shape[:2], -1)

    def keep(self, lengths, path):
        """Of the drafts after ``lengths`` those of ``path`` (node numbers, ascending) become the next tokens."""
        new = self.at(lengths[:, None] + torch.arange(path.shape[1], device=path.device))
        old = self.at(lengths[:, None] + path)
        self.k[new], self.v[new] = self.k[old], self.v[old]


class Stack(nn.Module):
    def __init__(self, layers=12, width=768, heads=12, vocabulary=50304, context=1024, latent_ratio=0.01, window=None,
                 sinks=0) -> None:
        super().__init__()
        self.heads = heads
        self.local = {} if window is None and not sinks else {"window": window, "sinks": sinks}
        self.tokens, self.positions = nn.Embedding(vocabulary, width), nn.Embedding(context, width)
        nn.init.normal_(self.tokens.weight, std=0.02)
        nn.init.normal_(self.positions.weight, std=0.02)
        self.blocks = nn.ModuleList(Block(width, heads, latent_ratio, i) for i in range(layers))
        self.norm = lwl.LayerNorm(width)

    def run(self, ids, positions, attends):
        delta, stream = self.positions(positions), self.tokens(ids)
        delta = delta.expand_as(stream)
        for block, attend in zip(self.blocks, attends):
            delta, stream = block(delta, stream, attend)
        return self.norm(delta, stream)[0]

    def forward(self, ids):
        """Logits of every position, for training."""
        attend = [lambda qkv: lwl.attention_packed(qkv, self.heads, **self.local)] * len(self.blocks)
        return F.linear(self.run(ids, torch.arange(ids.shape[1], device=ids.device), attend), self.tokens.weight)

    def step(self, ids, targets, optimizer):
        """One training step through the weight cache; returns the loss, the mean over the targets that are not padding
        (negative ones)."""
        optimizer.zero_grad(set_to_none=True)
        lwl.prepare_block_fht_weight_cache(self)
        loss = -lwl.token_log_probs(self(ids), targets).sum() / (targets >= 0).sum()
        loss.backward()
        lwl.flush_block_fht_weight_cache(self)
        optimizer.step()
        return loss.detach()

    def prompt(self, prompts, lengths, capacity):
        """The blocks' caches of ``prompts``, and the last tokens' features."""
        batch, tokens = prompts.shape
        caches = [Cache(batch, self.heads, capacity, self.norm.features // self.heads, self.tokens.weight, self.local)
                  for _ in self.blocks]
        x = self.run(prompts, torch.arange(tokens, device=prompts.device),
                     [lambda qkv, c=c: c.prompt(qkv, lengths) for c in caches])
        return caches, x[torch.arange(batch, device=x.device), lengths - 1]

    @torch.no_grad()
    def decode(self, prompts, lengths, new_tokens):
        """Greedy continuation of ``prompts`` (``[batch, tokens]``, padded at their ends to the longest of
        ``lengths``): ``(tokens, logits)``, ``[batch, new_tokens]`` and the logits that chose them."""
        lwl.prepare_block_fht_weight_cache(self)
        caches, x = self.prompt(prompts, lengths, prompts.shape[1] + new_tokens)
        chosen, scores = [], []
        for i in range(new_tokens):
            scores.append(F.linear(x, self.tokens.weight))
            chosen.append(scores[-1].argmax(-1))
            if i + 1 < new_tokens:
                at = lengths + i
                x = self.run(chosen[-1][:, None], at[:, None],
                             [lambda qkv, c=c: c.token(qkv, at) for c in caches])[:, 0]
        lwl.flush_block_fht_weight_cache(self)
        return torch.stack(chosen, 1), torch.stack(scores, 1)

    @torch.no_grad()
    def decode_drafts(self, prompts, lengths, new_tokens, draft):
        """The same tokens as ``decode``, several a pass: ``(tokens, log_probs, passes)``.

        ``draft(known)`` is given each sequence's tokens so far (lists) and returns a tree for each, ``(tokens,
        parents)`` of ``[batch, nodes]`` lists: node 0 is the last known token, every other node a guess of what follows
        its parent, two children of a node being different.  A pass computes all nodes; from node 0 on the path goes to the
        child that the model chooses as long as there is one, and every pass yields one more token than it has steps."""
        if self.local:
            raise ValueError("a tree of drafts sees its whole sequence, not a window of it")
        batch = len(prompts)
        known = [p[:n] for p, n in zip(prompts.tolist(), lengths.tolist())]
        ends = [len(k) + new_tokens for k in known]
        lwl.prepare_block_fht_weight_cache(self)
        caches, x = self.prompt(prompts, lengths, prompts.shape[1] + new_tokens + 128)
        nothing = torch.full((batch, 1), -1, device=x.device)
        _, best, chosen = lwl.token_log_probs(F.linear(x, self.tokens.weight), nothing, top=1)
        found = [[b] for b in best[:, 0].tolist()]
        for k, c in zip(known, chosen[:, 0].tolist()):
            k.append(c)
        passes = 0
        while any(len(k) < end for k, end in zip(known, ends)):
            tree, above = draft(known)
            children = [[[i for i, p in enumerate(above[b]) if p == n] for n in range(len(above[b]))] for b in range(batch)]
            depth = [[0] * len(t) for t in tree]
            for b in range(batch):
                for i, p in enumerate(above[b]):
                    depth[b][i] = depth[b][p] + 1 if p >= 0 else 0
            most = max(1, max(len(c) for nodes in children for c in nodes))
            asked = [[[tree[b][i] for i in c] + [-1] * (most - len(c)) for c in children[b]] for b in range(batch)]
            tokens, parents, deep, asked = (torch.tensor(t, device=x.device) for t in (tree, above, depth, asked))
            places = (lengths[:, None] + deep).clamp_max(self.positions.num_embeddings - 1)
            x = self.run(tokens, places, [lambda qkv, c=c: c.drafts(qkv, lengths, parents) for c in caches])
            of_drafts, best, chosen = lwl.token_log_probs(F.linear(x, self.tokens.weight), asked, top=1)
            of_drafts, best, chosen = of_drafts.tolist(), best[..., 0].tolist(), chosen[..., 0].tolist()
            paths, steps = [], []
            for b in range(batch):
                path, left = [0], ends[b] - len(known[b])
                while len(path) < left:
                    at = path[-1]
                    follows = [(n, i) for n, i in enumerate(children[b][at]) if tree[b][i] == chosen[b][at]]
                    if not follows:
                        break
                    found[b].append(of_drafts[b][at][follows[0][0]])
                    path.append(follows[0][1])
                if left > 0:
                    known[b] += [tree[b][i] for i in path[1:]] + [chosen[b][path[-1]]]
                    found[b].append(best[b][path[-1]])
                paths.append(path)
                steps.append(len(path) if left > 0 else 0)
            longest = max(len(p) for p in paths)
            path = torch.tensor([p + [p[-1]] * (longest - len(p)) for p in paths], device=x.device)
            for c in caches:
                c.keep(lengths, path)
            lengths = lengths + torch.tensor(steps, device=x.device)
            passes += 1
        lwl.flush_block_fht_weight_cache(self)
        new = [k[end - new_tokens:end] for k, end in zip(known, ends)]
        return torch.tensor(new), torch.tensor([f[:new_tokens] for f in found]), passes


def repeats(known, branches=4, depth=7):
    """Drafts from a sequence itself: what followed earlier occurrences of its last token."""
    trees = []
    for k in known:
        tokens, parents = [k[-1]], [-1]
        for at in [i for i in range(len(k) - 2, -1, -1) if k[i] == k[-1]][:branches]:
            node = 0
            for t in k[at + 1:at + 1 + depth]:
                same = [i for i in range(1, len(tokens)) if parents[i] == node and tokens[i] == t]
                if same:
                    node = same[0]
                else:
                    tokens.append(t)
                    parents.append(node)
                    node = len(tokens) - 1
        trees.append((tokens, parents))
    nodes = max(len(t) for t, _ in trees)
    # trees of one size: what is missing are roots of their own, which nobody follows
    pad = [(t + [0] * (nodes - len(t)), p + [-1] * (nodes - len(p))) for t, p in trees]
    return [t for t, _ in pad], [p for _, p in pad]


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--layers", type=int, default=12)
    p.add_argument("--batch", type=int, default=8)
    p.add_argument("--tokens", type=int, default=1024)
    p.add_argument("--steps", type=int, default=10)
    p.add_argument("--new-tokens", type=int, default=64)
    p.add_argument("--window", type=int, default=None, help="attend to this many last tokens only")
    p.add_argument("--sinks", type=int, default=0, help="and to these first ones")
    args = p.parse_args()
    torch.manual_seed(0)
    model = Stack(args.layers, context=args.tokens + args.new_tokens, window=args.window, sinks=args.sinks)
    model = model.cuda().bfloat16()
    optimizer = torch.optim.AdamW(model.parameters(), lr=1e-3, fused=True)
    ids = torch.randint(50304, (args.batch, args.tokens + 1), device="cuda")
    x, y = ids[:, :-1].contiguous(), ids[:, 1:].contiguous()

    def clock():
        torch.cuda.synchronize()
        return time.perf_counter()

    losses = [model.step(x, y, optimizer) for _ in range(3)]
    t = clock()
    losses += [model.step(x, y, optimizer) for _ in range(args.steps)]
    t = (clock() - t) / args.steps
    print(f"training: {1e3 * t:.2f} ms a step of {args.batch} x {args.tokens} tokens, loss {losses[0]:.3f} -> "
          f"{losses[-1]:.3f}, at most {torch.cuda.max_memory_allocated() / 2**30:.2f} GiB", flush=True)

    lengths = torch.linspace(args.tokens // 2, args.tokens, args.batch, device="cuda").long()
    model.decode(x, lengths, 3)
    spent = []
    for n in (1, args.new_tokens):
        t = clock()
        model.decode(x, lengths, n)
        spent.append(clock() - t)
    print(f"decoding: prompts {1e3 * spent[0]:.2f} ms, then {1e3 * (spent[1] - spent[0]) / max(args.new_tokens - 1, 1):.2f}"
          f" ms a token for {args.batch} sequences", flush=True)
    if not model.local:
        t = clock()
        passes = model.decode_drafts(x, lengths, args.new_tokens, repeats)[2]
        print(f"with drafts from the sequences themselves: {passes} passes for {args.new_tokens} tokens, "
              f"{1e3 * (clock() - t):.2f} ms", flush=True)


if __name__ == "__main__":
    main()
