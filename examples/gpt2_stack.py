"""A GPT-2 shaped stack of generated linears with the operators between them: a training step and decoding.

    python examples/gpt2_stack.py                      # 12 layers of 768, bfloat16: a training step, then decoding
    python examples/gpt2_stack.py --layers 2 --batch 2

The four linears of a block are ``BlockFHTLinear``s (reference ``examples/nanogpt/model.py``), used through
the weight cache: weights are generated once a step, and their gradients projected onto the latents
once.  Between them, each in one pass over its data: the residual addition with the layer norm, attention
straight from one linear's output to the next one's input, and the GELU that keeps 8 bits of its input.
Random weights and tokens.
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

    def __init__(self, batch, heads, capacity, head_size, like):
        self.k, self.v = (like.new_empty(batch, heads, capacity, head_size) for _ in range(2))

    def split(self, qkv):
        batch, tokens, _ = qkv.shape
        return qkv.view(batch, tokens, 3, self.k.shape[1], -1).permute(2, 0, 3, 1, 4)

    def prompt(self, qkv, lengths):
        """Attention of prompts padded at their ends, which become the cache's first tokens."""
        _, k, v = self.split(qkv)
        self.k[:, :, :qkv.shape[1]], self.v[:, :, :qkv.shape[1]] = k, v
        return lwl.attention_packed(qkv, self.k.shape[1], key_lengths=lengths, causal_offset=0)

    def token(self, qkv, lengths):
        """Attention of one new token for each sequence over what the cache holds of it and itself."""
        q, k, v = self.split(qkv)
        rows = torch.arange(len(lengths), device=lengths.device)
        self.k[rows, :, lengths], self.v[rows, :, lengths] = k[:, :, 0], v[:, :, 0]
        out = lwl.attention(q, self.k, self.v, key_lengths=lengths + 1)
        return out.transpose(1, 2).reshape(qkv.shape[0], 1, -1)


class Stack(nn.Module):
    def __init__(self, layers=12, width=768, heads=12, vocabulary=50304, context=1024, latent_ratio=0.01) -> None:
        super().__init__()
        self.heads = heads
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
        attend = [lambda qkv: lwl.attention_packed(qkv, self.heads)] * len(self.blocks)
        return F.linear(self.run(ids, torch.arange(ids.shape[1], device=ids.device), attend), self.tokens.weight)

    def step(self, ids, targets, optimizer):
        """One training step through the weight cache; returns the loss."""
        optimizer.zero_grad(set_to_none=True)
        lwl.prepare_block_fht_weight_cache(self)
        loss = F.cross_entropy(self(ids).flatten(0, 1).float(), targets.flatten())
        loss.backward()
        lwl.flush_block_fht_weight_cache(self)
        optimizer.step()
        return loss.detach()

    @torch.no_grad()
    def decode(self, prompts, lengths, new_tokens):
        """Greedy continuation of ``prompts`` (``[batch, tokens]``, padded at their ends to the longest of
        ``lengths``): ``(tokens, logits)``, ``[batch, new_tokens]`` and the logits that chose them."""
        batch, tokens = prompts.shape
        width = self.norm.features
        lwl.prepare_block_fht_weight_cache(self)
        caches = [Cache(batch, self.heads, tokens + new_tokens, width // self.heads, self.tokens.weight)
                  for _ in self.blocks]
        x = self.run(prompts, torch.arange(tokens, device=prompts.device),
                     [lambda qkv, c=c: c.prompt(qkv, lengths) for c in caches])
        x = x[torch.arange(batch, device=x.device), lengths - 1]
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


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--layers", type=int, default=12)
    p.add_argument("--batch", type=int, default=8)
    p.add_argument("--tokens", type=int, default=1024)
    p.add_argument("--steps", type=int, default=10)
    p.add_argument("--new-tokens", type=int, default=64)
    args = p.parse_args()
    torch.manual_seed(0)
    model = Stack(args.layers, context=args.tokens + args.new_tokens).cuda().bfloat16()
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


if __name__ == "__main__":
    main()
