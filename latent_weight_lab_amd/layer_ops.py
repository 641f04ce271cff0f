"""Tensor-level calls of the operators between a block's generated linears (``include/lwl_layers.h``):
layer norm, GELU with an 8-bit checkpoint, attention.

As in ``ops``: each function checks its arguments, allocates outputs and scratch through torch's
caching allocator and launches on the current stream of the tensors' device; nothing computes on
the CPU, and nothing here records gradients.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _native as N

GELU8_GROUP = 128


class LayerNormArgs(ctypes.Structure):
    """``lwl_layer_norm_args``."""
    _fields_ = [("dtype", ctypes.c_int32), ("weight_dtype", ctypes.c_int32), ("rows", ctypes.c_int64),
                ("features", ctypes.c_int64), ("eps", ctypes.c_double), ("x", ctypes.c_void_p),
                ("residual", ctypes.c_void_p), ("weight", ctypes.c_void_p), ("bias", ctypes.c_void_p),
                ("out", ctypes.c_void_p), ("sum", ctypes.c_void_p), ("stats", ctypes.c_void_p)]


class Gelu8Args(ctypes.Structure):
    """``lwl_gelu8_args``."""
    _fields_ = [("dtype", ctypes.c_int32), ("tanh_form", ctypes.c_int32), ("rows", ctypes.c_int64),
                ("features", ctypes.c_int64), ("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p)]


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
    i64, i32, sz, vp = ctypes.c_int64, ctypes.c_int, ctypes.c_size_t, ctypes.c_void_p
    normp, gelup, attnp = (ctypes.POINTER(t) for t in (LayerNormArgs, Gelu8Args, AttentionArgs))
    sigs = {
        "lwl_layer_norm_check": (i32, [normp]),
        "lwl_layer_norm_forward": (i32, [normp, vp]),
        "lwl_layer_norm_backward_workspace_size": (sz, [i64, i64]),
        "lwl_layer_norm_backward": (i32, [normp, vp, vp, vp, vp, vp, vp, sz, vp]),
        "lwl_gelu8_pitch": (i64, [i64]),
        "lwl_gelu8_check": (i32, [gelup]),
        "lwl_gelu8_forward": (i32, [gelup, vp, vp, vp, vp]),
        "lwl_gelu8_activation": (i32, [gelup, vp, vp]),
        "lwl_gelu8_backward_workspace_size": (sz, [i64, i64]),
        "lwl_gelu8_backward": (i32, [gelup, vp, vp, vp, vp, sz, vp]),
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


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------- layer norm
def _check_vector(name: str, t: torch.Tensor, n: int, dtype: torch.dtype) -> torch.Tensor:
    if t.dim() != 1 or t.numel() != n or t.dtype != dtype:
        raise N.BlockFHTArgumentError(f"{name} must be {n} values of {dtype}, got {tuple(t.shape)} of {t.dtype}")
    return t.contiguous()


def _norm_args(x: torch.Tensor, weight: torch.Tensor, eps: float, rows: int) -> LayerNormArgs:
    a = LayerNormArgs()
    a.dtype, a.weight_dtype = N.dtype_code(x.dtype), N.dtype_code(weight.dtype)
    a.rows, a.features, a.eps = rows, int(x.shape[-1]), float(eps)
    return a


def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, eps: float,
                       residual: torch.Tensor | None, keep_stats: bool):
    """``(out, sum, stats)`` over the last dimension of x; ``sum`` is None without a residual, ``stats``
    (float32 ``[2, rows]``: means, reciprocal deviations) unless ``keep_stats``."""
    if x.dim() < 1 or x.shape[-1] == 0:
        raise N.BlockFHTArgumentError("layer norm needs at least one feature")
    dev = N.require_cuda(x, weight, *[t for t in (bias, residual) if t is not None])
    features = int(x.shape[-1])
    a = _norm_args(x, weight, eps, x.numel() // features)
    L = N.lib()
    N.check(L.lwl_layer_norm_check(ctypes.byref(a)))
    weight = _check_vector("layer norm's weight", weight, features, weight.dtype)
    if bias is not None:
        bias = _check_vector("layer norm's bias", bias, features, weight.dtype)
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise N.BlockFHTArgumentError(
                f"residual must be {tuple(x.shape)} of {x.dtype}, got {tuple(residual.shape)} of {residual.dtype}")
        residual = residual.contiguous()
    x = x.contiguous()
    out = torch.empty_like(x)
    total = torch.empty_like(x) if residual is not None else None
    stats = torch.empty(2, a.rows, dtype=torch.float32, device=dev) if keep_stats else None
    a.x, a.residual, a.weight, a.bias = _ptr(x), _ptr(residual), _ptr(weight), _ptr(bias)
    a.out, a.sum, a.stats = _ptr(out), _ptr(total), _ptr(stats)
    with torch.cuda.device(dev):
        N.check(L.lwl_layer_norm_forward(ctypes.byref(a), N.stream_ptr(dev)))
    return out, total, stats


def layer_norm_backward(h: torch.Tensor, weight: torch.Tensor, stats: torch.Tensor, eps: float, grad_out: torch.Tensor,
                        grad_sum: torch.Tensor | None, need_x: bool, need_weight: bool, need_bias: bool):
    """``(grad_x, grad_weight, grad_bias)``, None for what is not needed; ``h`` is what was normed."""
    dev = N.require_cuda(h, weight, stats, grad_out)
    features = int(h.shape[-1])
    a = _norm_args(h, weight, eps, h.numel() // features)
    L = N.lib()
    N.check(L.lwl_layer_norm_check(ctypes.byref(a)))
    grad_out = grad_out.to(h.dtype).contiguous()
    grad_sum = None if grad_sum is None else grad_sum.to(h.dtype).contiguous()
    gx = torch.empty_like(h) if need_x else None
    gw = torch.empty(features, dtype=weight.dtype, device=dev) if need_weight else None
    gb = torch.empty(features, dtype=weight.dtype, device=dev) if need_bias else None
    a.x, a.weight, a.stats = _ptr(h), _ptr(weight), _ptr(stats)
    with torch.cuda.device(dev):
        need = L.lwl_layer_norm_backward_workspace_size(a.rows, a.features) if need_weight or need_bias else 0
        ws_ptr, ws_size, ws = N.workspace(need, dev)
        N.check(L.lwl_layer_norm_backward(ctypes.byref(a), _ptr(grad_out), _ptr(grad_sum), _ptr(gx), _ptr(gw),
                                          _ptr(gb), ws_ptr, ws_size, N.stream_ptr(dev)))
    del ws
    return gx, gw, gb


# ---------------------------------------------------------------- GELU, input kept in 8 bits
_FORMS = {"none": 0, "tanh": 1}


def _gelu8_args(dtype: torch.dtype, rows: int, features: int, approximate: str) -> Gelu8Args:
    if approximate not in _FORMS:
        raise N.BlockFHTArgumentError(f"approximate must be 'none' or 'tanh', got {approximate!r}")
    a = Gelu8Args()
    a.dtype, a.tanh_form, a.rows, a.features = N.dtype_code(dtype), _FORMS[approximate], rows, features
    return a


def gelu8_forward(x: torch.Tensor, bias: torch.Tensor | None, approximate: str, keep: bool):
    """``(gelu(x + bias), codes, scales)`` over the last dimension of x; codes (int8 ``[rows, pitch]``) and
    scales (float32 ``[rows, groups]``) are None unless ``keep``."""
    if x.dim() < 1 or x.shape[-1] == 0:
        raise N.BlockFHTArgumentError("GELU checkpoint needs at least one feature")
    dev = N.require_cuda(x, *[t for t in (bias,) if t is not None])
    features = int(x.shape[-1])
    rows = x.numel() // features
    a = _gelu8_args(x.dtype, rows, features, approximate)
    L = N.lib()
    N.check(L.lwl_gelu8_check(ctypes.byref(a)))
    if bias is not None:
        bias = _check_vector("GELU's bias", bias, features, x.dtype)
    x = x.contiguous()
    out = torch.empty_like(x)
    codes = scales = None
    if keep:
        codes = torch.empty(rows, (features + 7) // 8 * 8, dtype=torch.int8, device=dev)
        scales = torch.empty(rows, -(-features // GELU8_GROUP), dtype=torch.float32, device=dev)
        a.codes, a.scales = _ptr(codes), _ptr(scales)
    with torch.cuda.device(dev):
        N.check(L.lwl_gelu8_forward(ctypes.byref(a), _ptr(x), _ptr(bias), _ptr(out), N.stream_ptr(dev)))
    return out, codes, scales


def gelu8_activation(codes: torch.Tensor, scales: torch.Tensor, shape: tuple[int, ...], dtype: torch.dtype,
                     approximate: str) -> torch.Tensor:
    """``gelu`` of what the checkpoint stands for, in ``shape`` and ``dtype``."""
    dev = N.require_cuda(codes, scales)
    out = torch.empty(shape, dtype=dtype, device=dev)
    a = _gelu8_args(dtype, codes.shape[0], int(shape[-1]), approximate)
    a.codes, a.scales = _ptr(codes), _ptr(scales)
    with torch.cuda.device(dev):
        N.check(N.lib().lwl_gelu8_activation(ctypes.byref(a), _ptr(out), N.stream_ptr(dev)))
    return out


def gelu8_backward(codes: torch.Tensor, scales: torch.Tensor, grad_out: torch.Tensor, dtype: torch.dtype,
                   approximate: str, need_bias: bool):
    """``(grad_x, grad_bias)``; ``grad_out`` has the activation's shape."""
    dev = N.require_cuda(codes, scales, grad_out)
    grad_out = grad_out.to(dtype).contiguous()
    features = int(grad_out.shape[-1])
    a = _gelu8_args(dtype, codes.shape[0], features, approximate)
    a.codes, a.scales = _ptr(codes), _ptr(scales)
    gx = torch.empty_like(grad_out)
    gb = torch.empty(features, dtype=dtype, device=dev) if need_bias else None
    L = N.lib()
    with torch.cuda.device(dev):
        need = L.lwl_gelu8_backward_workspace_size(a.rows, a.features) if need_bias else 0
        ws_ptr, ws_size, ws = N.workspace(need, dev)
        N.check(L.lwl_gelu8_backward(ctypes.byref(a), _ptr(grad_out), _ptr(gx), _ptr(gb), ws_ptr, ws_size,
                                     N.stream_ptr(dev)))
    del ws
    return gx, gb


# ---------------------------------------------------------------- attention
ATTENTION_MAX_DIM = 128


def _dense_dim(t: torch.Tensor) -> torch.Tensor:
    # the kernels take any strides but that of a head's values, which lie one after the other
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def _strides(t: torch.Tensor) -> _Strides:
    return _Strides(t.stride(0), t.stride(1), t.stride(2))


def _attention_args(q, k, v, causal, scale, key_lengths, causal_offset) -> tuple[AttentionArgs, list]:
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4:
            raise N.BlockFHTArgumentError(f"attention: {name} must be [batch, heads, tokens, head size], got {tuple(t.shape)}")
    if k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise N.BlockFHTArgumentError(f"attention: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not match")
    if not q.dtype == k.dtype == v.dtype:
        raise N.BlockFHTArgumentError(f"attention: q, k and v must have one type, got {q.dtype}, {k.dtype} and {v.dtype}")
    a = AttentionArgs()
    a.dtype, a.causal = N.dtype_code(q.dtype), int(bool(causal))
    a.bottom_right, a.causal_offset = int(causal_offset is None), int(causal_offset or 0)
    a.batch, a.heads, a.queries, a.dim = q.shape
    a.kv_heads, a.keys = int(k.shape[1]), int(k.shape[2])
    a.scale = 1.0 / math.sqrt(max(1, a.dim)) if scale is None else float(scale)
    N.check(N.lib().lwl_attention_check(ctypes.byref(a)))
    keep = [_dense_dim(t.detach()) for t in (q, k, v)]
    a.q, a.k, a.v = (_ptr(t) for t in keep)
    a.q_stride, a.k_stride, a.v_stride = (_strides(t) for t in keep)
    if key_lengths is not None:
        if key_lengths.dim() != 1 or key_lengths.numel() != a.batch or key_lengths.is_floating_point():
            raise N.BlockFHTArgumentError(f"attention: key_lengths must be {a.batch} integers, got {tuple(key_lengths.shape)}"
                                          f" of {key_lengths.dtype}")
        lengths = key_lengths.to(torch.int32).contiguous()
        a.key_lengths = _ptr(lengths)
        keep.append(lengths)
    return a, keep


def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool, scale: float | None,
                      key_lengths: torch.Tensor | None, causal_offset: int | None, keep_lse: bool,
                      out: torch.Tensor | None = None):
    """``(out, lse)`` for ``[batch, heads, tokens, head size]`` tensors; ``out`` lies in memory token by token
    (all heads of a token together); ``lse`` (float32 ``[batch, heads, queries]``) is None unless ``keep_lse``."""
    dev = N.require_cuda(q, k, v, *[t for t in (key_lengths,) if t is not None])
    a, keep = _attention_args(q, k, v, causal, scale, key_lengths, causal_offset)
    if out is None:
        out = torch.empty(a.batch, a.queries, a.heads, a.dim, dtype=q.dtype, device=dev).transpose(1, 2)
    lse = torch.empty(a.batch, a.heads, a.queries, dtype=torch.float32, device=dev) if keep_lse else None
    a.out, a.lse, a.out_stride = _ptr(out), _ptr(lse), _strides(out)
    L = N.lib()
    with torch.cuda.device(dev):
        ws_ptr, ws_size, ws = N.workspace(L.lwl_attention_forward_workspace_size(ctypes.byref(a)), dev)
        N.check(L.lwl_attention_forward(ctypes.byref(a), ws_ptr, ws_size, N.stream_ptr(dev)))
    del ws, keep
    return out, lse


def attention_backward(q, k, v, out, lse, grad_out, causal, scale, key_lengths, causal_offset, grads):
    """Fills ``grads``, the three gradients like q, k and v (any strides, a head's values dense)."""
    dev = N.require_cuda(q, k, v, out, lse, grad_out)
    a, keep = _attention_args(q, k, v, causal, scale, key_lengths, causal_offset)
    grad_out = _dense_dim(grad_out.to(q.dtype))
    a.out, a.lse, a.grad_out = _ptr(out), _ptr(lse), _ptr(grad_out)
    a.out_stride, a.grad_out_stride = _strides(out), _strides(grad_out)
    a.grad_q, a.grad_k, a.grad_v = (_ptr(t) for t in grads)
    a.grad_q_stride, a.grad_k_stride, a.grad_v_stride = (_strides(t) for t in grads)
    L = N.lib()
    with torch.cuda.device(dev):
        ws_ptr, ws_size, ws = N.workspace(L.lwl_attention_backward_workspace_size(ctypes.byref(a)), dev)
        N.check(L.lwl_attention_backward(ctypes.byref(a), ws_ptr, ws_size, N.stream_ptr(dev)))
    del ws, keep
