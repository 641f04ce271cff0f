"""Tensor-level calls of the operators between a block's generated linears (``include/lwl_layers.h``):
layer norm, GELU with an 8-bit checkpoint, attention.

The calls go through the torch binding ``lib/lwl_layers.so`` (``csrc/torch_ext``), which checks arguments,
allocates through torch's caching allocator, launches on the current stream of the tensors' device and
records gradients in C++.  Nothing computes on the CPU.  The C entries' ctypes signatures are here too.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native as N

GELU8_GROUP = 128

_Strides = ctypes.c_int64 * 3


class AttentionArgs(ctypes.Structure):
    """``lwl_attention_args``."""
    _fields_ = [("dtype", ctypes.c_int32), ("causal", ctypes.c_int32), ("bottom_right", ctypes.c_int32),
                ("reserved", ctypes.c_int32), ("causal_offset", ctypes.c_int64), ("batch", ctypes.c_int64),
                ("heads", ctypes.c_int64), ("kv_heads", ctypes.c_int64), ("queries", ctypes.c_int64),
                ("keys", ctypes.c_int64), ("dim", ctypes.c_int64), ("scale", ctypes.c_double),
                ("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("out", ctypes.c_void_p),
                ("lse", ctypes.c_void_p), ("key_lengths", ctypes.c_void_p), ("q_stride", _Strides),
                ("k_stride", _Strides), ("v_stride", _Strides), ("out_stride", _Strides),
                ("grad_out", ctypes.c_void_p), ("grad_q", ctypes.c_void_p), ("grad_k", ctypes.c_void_p),
                ("grad_v", ctypes.c_void_p), ("grad_out_stride", _Strides), ("grad_q_stride", _Strides),
                ("grad_k_stride", _Strides), ("grad_v_stride", _Strides)]


def bind(lib) -> None:
    """Signatures of ``lwl_layers.h`` on the loaded library."""
    i64, i32, sz, vp, dbl = ctypes.c_int64, ctypes.c_int, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_double
    attnp = ctypes.POINTER(AttentionArgs)
    sigs = {
        "lwl_layer_norm_check": (i32, [i32, i32, i64, i64, dbl]),
        "lwl_layer_norm_forward": (i32, [vp, vp, vp, vp, i32, i32, i64, i64, dbl, vp, vp, vp, vp]),
        "lwl_layer_norm_backward_workspace_size": (sz, [i64, i64]),
        "lwl_layer_norm_backward": (i32, [vp, vp, vp, vp, vp, i32, i32, i64, i64, vp, vp, vp, vp, sz, vp]),
        "lwl_gelu8_pitch": (i64, [i64]),
        "lwl_gelu8_check": (i32, [i32, i64, i64]),
        "lwl_gelu8_forward": (i32, [vp, vp, i32, i32, i64, i64, vp, vp, vp, vp]),
        "lwl_gelu8_activation": (i32, [vp, vp, i32, i32, i64, i64, vp, vp]),
        "lwl_gelu8_backward_workspace_size": (sz, [i64, i64]),
        "lwl_gelu8_backward": (i32, [vp, vp, vp, i32, i32, i64, i64, vp, vp, vp, sz, vp]),
        "lwl_attention_check": (i32, [attnp]),
        "lwl_attention_forward_workspace_size": (sz, [attnp]),
        "lwl_attention_forward": (i32, [attnp, vp, sz, vp]),
        "lwl_attention_backward_workspace_size": (sz, [attnp]),
        "lwl_attention_backward": (i32, [attnp, vp, sz, vp]),
    }
    for name, (res, args) in sigs.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args


_FORMS = {"none": False, "tanh": True}


def tanh_form(approximate: str) -> bool:
    if approximate not in _FORMS:
        raise N.BlockFHTArgumentError(f"approximate must be 'none' or 'tanh', got {approximate!r}")
    return _FORMS[approximate]


def gelu8_activation(codes: torch.Tensor, scales: torch.Tensor, shape: tuple[int, ...], dtype: torch.dtype,
                     approximate: str) -> torch.Tensor:
    """``gelu`` of what the checkpoint stands for, in ``shape`` and ``dtype``."""
    return N.layers().gelu8_activation(codes, scales, shape, dtype, tanh_form(approximate))


def gelu8_backward(codes: torch.Tensor, scales: torch.Tensor, grad_out: torch.Tensor, dtype: torch.dtype,
                   approximate: str, need_bias: bool):
    """``(grad_x, grad_bias)`` in ``dtype``; ``grad_out`` has the activation's shape."""
    return N.layers().gelu8_backward(codes, scales, grad_out, dtype, tanh_form(approximate), need_bias)


def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool, scale: float | None,
                      key_lengths: torch.Tensor | None, causal_offset: int | None, keep_lse: bool,
                      window: int | None = None, sinks: int = 0):
    """``(out, lse)`` for ``[batch, heads, tokens, head size]`` tensors; ``out`` lies in memory token by token
    (all heads of a token together); ``lse`` (float32 ``[batch, heads, queries]``) is None unless ``keep_lse``."""
    return N.layers().attention_forward(q, k, v, causal, scale, key_lengths, causal_offset, keep_lse, window, sinks)


def attention_backward(q, k, v, out, lse, grad_out, causal, scale, key_lengths, causal_offset, window=None, sinks=0):
    """The gradients of q, k and v; each lies in memory token by token, as ``out``."""
    return N.layers().attention_backward(q, k, v, out, lse, grad_out, causal, scale, key_lengths, causal_offset, window,
                                         sinks)
