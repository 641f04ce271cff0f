"""Log probabilities of given tokens, with the entropy and the most probable alternatives: a training loss, and what
sampled or drafted tokens are judged by.

The reference's model calls torch's cross entropy (``examples/nanogpt/model.py``).  Here the forward is one pass over the
logits in their own type and the backward one more, which writes their gradient (``lwl_log_probs_forward`` /
``_backward``); nothing of the logits' size is kept beside the logits.
"""
from __future__ import annotations

import torch

from . import _native as N


def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor, entropy: bool = False,
                    top: int = 0) -> torch.Tensor | tuple[torch.Tensor, ...]:
    """``log softmax(logits)`` of ``tokens``.

    ``logits`` is ``[..., vocabulary]`` in float32, float16 or bfloat16; rows may lie apart (slices of padded or shifted
    rows are read where they are).  ``tokens`` are integers of the leading shape, or with one more axis of up to 64
    tokens of each row; the result is float32 in their shape.  A negative token stands for none (padding): 0, without a
    gradient.  One past the vocabulary gives NaN, without a gradient.  A loss over padded targets is their sum
    divided by the number that is there, ``-token_log_probs(logits, targets).sum() / (targets >= 0).sum()``.

    With ``entropy`` or ``top`` the result is a tuple: the log probabilities; with ``entropy`` ``-sum p log p`` of every row;
    with ``top`` (up to 64) the largest log probabilities, ``[..., top]`` in descending order, and their tokens (int64).
    Of equal logits the lowest token comes first.

    Differentiable in the logits (once, in reverse mode), through all three; the gradient is contiguous and in the
    logits' type.  Sums are float32.  Logits of minus infinity are tokens of probability 0; a row of nothing else has log
    probabilities of minus infinity, entropy 0, the first tokens on top and no gradient.  A NaN or plus infinity makes
    its row's results NaN."""
    out = N.layers().token_log_probs(logits, tokens, entropy, top)
    return tuple(out) if entropy or top else out[0]
