"""Layer norm over the last dimension, with the residual stream's addition in front of it.

The reference's model norms through torch (``examples/nanogpt/model.py``); here one HIP launch reads each
stream once, adds the residual, norms, and stores both (``lwl_layer_norm_forward``), and the
backward pass is one launch for the rows and one for the weight's and bias's sums.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _native as N


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, eps: float = 1e-5,
               residual: torch.Tensor | None = None):
    """``(h - mean(h)) / sqrt(var(h) + eps) * weight + bias`` over the last dimension of ``x``.

    Without ``residual`` h is x, and the normed tensor is returned.  With it h is ``x + residual``, rounded
    to x's type, and ``(normed, h)`` is returned: h is the residual stream that goes on.  ``x`` is
    float32, float16 or bfloat16; ``weight`` and ``bias`` have its type or are float32; mean, variance
    and the gradients' sums are float32.  Differentiable in all four tensors (once, in reverse mode)."""
    out = N.layers().layer_norm(x, weight, bias, eps, residual)
    return out[0] if residual is None else (out[0], out[1])


class LayerNorm(nn.Module):
    """Layer norm with an optional bias, as the reference model's norm; ``forward(x, residual)`` adds
    the residual first and returns the sum as well."""

    def __init__(self, features: int, bias: bool = True, eps: float = 1e-5) -> None:
        super().__init__()
        self.features, self.eps = int(features), float(eps)
        self.weight = nn.Parameter(torch.ones(self.features))
        self.bias = nn.Parameter(torch.zeros(self.features)) if bias else None

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        return layer_norm(x, self.weight, self.bias, self.eps, residual)
