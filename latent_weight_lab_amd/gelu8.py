"""GELU that keeps its input in 8 bits for the backward pass.

A generated linear stores no weight; what a training step then holds is activations.  The MLP's
hidden ones are the largest: in a 16-bit type GELU's input and its output (the next linear's input,
needed for that weight's gradient) take 4 bytes an element.  ``gelu_checkpoint8`` keeps the input as
8-bit codes with a float32 scale for 128 features (1.03 bytes), ``gelu_linear_checkpoint8`` lets the next
linear's gradient take its input from the same codes, so that the activation is not kept at all.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _native as N
from . import layer_ops


class Checkpoint8:
    """What is kept of GELU's input z: int8 ``codes``, float32 ``scales`` for groups of 128 features;
    they stand for ``codes * scale``."""

    def __init__(self, codes, scales, x, approximate):
        self.codes, self.scales = codes, scales
        self.shape, self.dtype, self.approximate = tuple(x.shape), x.dtype, approximate

    def values(self) -> torch.Tensor:
        """What the codes stand for, in float32 and the input's shape."""
        features = self.shape[-1]
        scale = self.scales.repeat_interleave(layer_ops.GELU8_GROUP, dim=1)[:, :features]
        return (self.codes[:, :features].float() * scale).reshape(self.shape)

    def activation(self) -> torch.Tensor:
        """GELU of what the codes stand for, in the input's type and shape."""
        return layer_ops.gelu8_activation(self.codes, self.scales, self.shape, self.dtype, self.approximate)

    def nbytes(self) -> int:
        return self.codes.numel() + 4 * self.scales.numel()


def gelu_checkpoint8(x: torch.Tensor, bias: torch.Tensor | None = None, approximate: str = "none",
                     return_checkpoint: bool = False):
    """``gelu(x + bias)`` over any leading dimensions; ``approximate`` as ``torch.nn.functional.gelu``'s.

    The forward value is exact (float32, rounded once); the backward pass takes the derivative at
    the 8-bit checkpoint of ``x + bias``.  With ``return_checkpoint`` returns ``(activation,
    Checkpoint8)``.  Where no gradient is recorded and no checkpoint asked for, nothing is kept.
    Differentiable once, in reverse mode; ``bias`` has x's type."""
    out, codes, scales = N.layers().gelu8(x, bias, layer_ops.tanh_form(approximate), return_checkpoint)
    return (out, Checkpoint8(codes, scales, x, approximate)) if return_checkpoint else out


def gelu_linear_checkpoint8(x: torch.Tensor, linear: nn.Module, bias: torch.Tensor | None = None,
                            approximate: str = "none") -> torch.Tensor:
    """``linear(gelu(x + bias))`` that keeps 1.03 bytes of each hidden element.

    What ``linear`` (a ``BlockFHTLinear``, cached or not, or any other module) saves of its input for the
    backward pass is replaced by the checkpoint and computed again from it there; the weight's (or
    latent's) gradient is then that of the checkpoint's activation.  What it saves of its input after
    changing it in place (a dropout with ``inplace=True``, say) is kept as it is.  Saved-tensor hooks around the
    call (offloading to the host) see the codes and scales, not what ``linear`` saves: hooks of torch do not
    nest.
    """
    if not torch.is_grad_enabled():
        return linear(gelu_checkpoint8(x, bias, approximate))
    y, checkpoint = gelu_checkpoint8(x, bias, approximate, return_checkpoint=True)
    span = (y.data_ptr(), y.numel(), y.dtype, y._version)

    def pack(t):
        # the activation itself or a dense view of all of it (flattened rows), not written to since: views
        # count their base's changes
        if t.is_cuda and (t.data_ptr(), t.numel(), t.dtype, t._version) == span and t.is_contiguous() and t.numel():
            return tuple(t.shape)
        return t

    def unpack(kept):
        return checkpoint.activation().view(kept) if isinstance(kept, tuple) else kept

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        return linear(y)
