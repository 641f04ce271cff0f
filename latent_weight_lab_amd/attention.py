"""Attention over the heads that the generated linears make, forward and backward, and over a cache.

The reference's model calls torch's attention (``examples/nanogpt/model.py``).  Here the forward is one pass
over the keys on the matrix cores, for prompts and for single tokens alike (few queries over a long cache
split the keys among workgroups), and the backward computes the probabilities again from the saved log
sums (``lwl_attention_forward`` / ``_backward``).  Nothing of size queries x keys is stored, and
gradients do not depend on the order in which workgroups run.
"""
from __future__ import annotations

import torch

from . import _native as N
from . import layer_ops


class _AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, key_lengths, causal, scale, causal_offset):
        out, lse = layer_ops.attention_forward(q, k, v, causal, scale, key_lengths, causal_offset, True)
        ctx.save_for_backward(q, k, v, out, lse, key_lengths)
        ctx.meta = (causal, scale, causal_offset)
        return out

    @staticmethod
    @layer_ops.once
    def backward(ctx, grad_out):
        q, k, v, out, lse, lengths = ctx.saved_tensors
        causal, scale, offset = ctx.meta
        # token by token in memory, as the linears before them leave q, k and v
        b, hq, tq, d = q.shape
        hk, tk = k.shape[1], k.shape[2]
        dtype, dev = q.dtype, q.device
        grads = (torch.empty((b, tq, hq, d), dtype=dtype, device=dev).transpose(1, 2),
                 torch.empty((b, tk, hk, d), dtype=dtype, device=dev).transpose(1, 2),
                 torch.empty((b, tk, hk, d), dtype=dtype, device=dev).transpose(1, 2))
        layer_ops.attention_backward(q, k, v, out, lse, grad_out, causal, scale, lengths, offset, grads)
        return (*grads, None, None, None, None)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = False, scale: float | None = None,
              key_lengths: torch.Tensor | None = None, causal_offset: int | None = None) -> torch.Tensor:
    """``softmax(scale * q k^T) v`` for each head.

    ``q`` is ``[batch, heads, queries, head size]``, ``k`` and ``v`` ``[batch, kv_heads, keys, head size]``; ``heads`` is a
    multiple of ``kv_heads``, and consecutive query heads share a key head.  Head sizes up to 128;
    float32, float16 or bfloat16; any strides (a head's values are made dense if they are not).
    ``scale`` defaults to ``1 / sqrt(head size)`` and must be positive.

    ``key_lengths`` (integers on the device, ``[batch]``): keys of each sequence; what lies past them in k and
    v is not read into any result (a cache's unused end).  ``causal``: query i sees keys up to
    ``i + causal_offset``; by default the queries are the last tokens of their sequence (offset ``length -
    queries``), so the same call serves a prompt (as many queries as keys), new tokens over a cache and
    one token.  A batch padded at its end trains with ``causal_offset=0``.

    A query that sees no key gives zeros and takes no part in the gradients.  The result is
    ``[batch, heads, queries, head size]`` and lies token by token in memory, so that
    ``out.transpose(1, 2).reshape(batch, queries, -1)`` copies nothing.  Softmax and sums are float32; in 16-bit
    types the probabilities are rounded to the type before the product with v.  Differentiable in q, k
    and v (once)."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _AttentionFn.apply(q, k, v, key_lengths, bool(causal), scale, causal_offset)
    return layer_ops.attention_forward(q, k, v, causal, scale, key_lengths, causal_offset, False)[0]


class _PackedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, heads, kv_heads, key_lengths, causal, scale, causal_offset):
        out, lse = layer_ops.attention_packed_forward(qkv, heads, kv_heads, causal, scale, key_lengths, causal_offset, True)
        ctx.save_for_backward(qkv, out, lse, key_lengths)
        ctx.meta = (heads, kv_heads, causal, scale, causal_offset)
        return out

    @staticmethod
    @layer_ops.once
    def backward(ctx, grad_out):
        qkv, out, lse, lengths = ctx.saved_tensors
        heads, kv_heads, causal, scale, offset = ctx.meta
        grad = layer_ops.attention_packed_backward(qkv, out, lse, grad_out, heads, kv_heads, causal, scale, lengths, offset)
        return grad, None, None, None, None, None, None


def attention_packed(qkv: torch.Tensor, heads: int, kv_heads: int | None = None, causal: bool = True,
                     scale: float | None = None, key_lengths: torch.Tensor | None = None,
                     causal_offset: int | None = None) -> torch.Tensor:
    """Self-attention straight from and to a block's linears: ``qkv`` is ``[batch, tokens, (heads + 2 kv_heads) *
    head size]``, queries, keys and values side by side (one linear's output), and the result ``[batch,
    tokens, heads * head size]``.  Nothing is split or copied, and the gradient is one tensor like qkv.  The
    other arguments are ``attention``'s."""
    heads = int(heads)
    kv_heads = heads if kv_heads is None else int(kv_heads)
    if qkv.dim() != 3 or heads <= 0 or kv_heads <= 0 or qkv.shape[2] % (heads + 2 * kv_heads):
        raise N.BlockFHTArgumentError(f"attention_packed: {tuple(qkv.shape)} does not hold {heads} query and twice "
                                      f"{kv_heads} key heads")
    if not qkv.is_contiguous():
        qkv = qkv.contiguous()
    if torch.is_grad_enabled() and qkv.requires_grad:
        return _PackedFn.apply(qkv, heads, kv_heads, key_lengths, bool(causal), scale, causal_offset)
    return layer_ops.attention_packed_forward(qkv, heads, kv_heads, causal, scale, key_lengths, causal_offset, False)[0]
