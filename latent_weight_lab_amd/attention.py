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


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = False, scale: float | None = None,
              key_lengths: torch.Tensor | None = None, causal_offset: int | None = None) -> torch.Tensor:
    """``softmax(scale * q k^T) v`` for each head.

    ``q`` is ``[batch, heads, queries, head size]``, ``k`` and ``v`` ``[batch, kv_heads, keys, head size]``; ``heads`` is a
    multiple of ``kv_heads``, and consecutive query heads share a key head.  Head sizes up to 128;
    float32, float16 or bfloat16; any strides (a head's values are made dense if they are not).
    ``scale`` defaults to ``1 / sqrt(head size)`` and must be positive (from 2^-100 to 2^100).

    ``key_lengths`` (integers on the device, ``[batch]``): keys of each sequence; what lies past them in k and
    v is not read into any result (a cache's unused end).  ``causal``: query i sees keys up to
    ``i + causal_offset``; by default the queries are the last tokens of their sequence (offset ``length -
    queries``), so the same call serves a prompt (as many queries as keys), new tokens over a cache and
    one token.  A batch padded at its end trains with ``causal_offset=0``.

    A query that sees no key gives zeros and takes no part in the gradients.  The result is
    ``[batch, heads, queries, head size]`` and lies token by token in memory, so that
    ``out.transpose(1, 2).reshape(batch, queries, -1)`` copies nothing.  Softmax and sums are float32; in 16-bit
    types the probabilities are rounded to the type before the product with v, and in the backward pass the
    probabilities and the scores' gradients before theirs.  Differentiable in q, k and v (once, in reverse mode).

    A NaN in a key or value that some query sees may also reach queries from which ``causal`` hides it, as where
    a masked score matrix is multiplied out, and one in a query or its gradient the gradients of keys hidden from it;
    float32 infinities in k, q or v give NaN."""
    return N.layers().attention(q, k, v, causal, scale, key_lengths, causal_offset)


def attention_packed(qkv: torch.Tensor, heads: int, kv_heads: int | None = None, causal: bool = True,
                     scale: float | None = None, key_lengths: torch.Tensor | None = None,
                     causal_offset: int | None = None) -> torch.Tensor:
    """Self-attention straight from and to a block's linears: ``qkv`` is ``[batch, tokens, (heads + 2 kv_heads) *
    head size]``, queries, keys and values side by side (one linear's output), and the result ``[batch,
    tokens, heads * head size]``.  Nothing is split or copied, and the gradient is one tensor like qkv.  The
    other arguments are ``attention``'s, but for ``causal_offset``: queries and keys are the same tokens, so it
    defaults to 0, also in a batch padded at its ends (``key_lengths``)."""
    return N.layers().attention_packed(qkv, heads, heads if kv_heads is None else kv_heads, causal, scale, key_lengths,
                                       causal_offset)
