"""Layer norm over the last dimension, with the residual stream's addition in front of it.

The reference's model norms through torch (``examples/nanogpt/model.py``); here one HIP launch reads each
stream once, adds the residual, norms, and stores both (``lwl_layer_norm_forward``), and the
backward pass is one launch for the rows and one for the weight's and bias's sums.
"""
from __future__ import annotations

import torch
from torch import nn

from . import layer_ops


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        out, total, stats = layer_ops.layer_norm_forward(x, weight, bias, eps, residual, True)
        h = total if total is not None else x.contiguous()
        ctx.save_for_backward(h, weight, stats)
        ctx.set_materialize_grads(False)
        return (out, total) if total is not None else out

    @staticmethod
    @layer_ops.once
    def backward(ctx, grad_out, grad_sum=None):
        h, weight, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        if grad_out is None:  # only the sum was used
            return (grad_sum if need[0] else None), (grad_sum if need[1] else None), None, None, None
        gx, gw, gb = layer_ops.layer_norm_backward(h, weight, stats, grad_out, grad_sum, need[0] or need[1],
                                                   need[2], need[3])
        return (gx if need[0] else None), (gx if need[1] else None), gw, gb, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, eps: float = 1e-5,
               residual: torch.Tensor | None = None):
    """``(h - mean(h)) / sqrt(var(h) + eps) * weight + bias`` over the last dimension of ``x``.

    Without ``residual`` h is x, and the normed tensor is returned.  With it h is ``x + residual``, rounded
    to x's type, and ``(normed, h)`` is returned: h is the residual stream that goes on.  ``x`` is
    float32, float16 or bfloat16; ``weight`` and ``bias`` have its type or are float32; mean, variance
    and the gradients' sums are float32.  Differentiable in all four tensors."""
    needs = [t for t in (x, residual, weight, bias) if t is not None and t.requires_grad]
    if torch.is_grad_enabled() and needs:
        return _LayerNormFn.apply(x, residual, weight, bias, float(eps))
    out, total, _ = layer_ops.layer_norm_forward(x, weight, bias, float(eps), residual, False)
    return out if residual is None else (out, total)


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
