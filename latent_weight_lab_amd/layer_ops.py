"""Tensor-level calls of the operators between a block's generated linears (``include/lwl_layers.h``):
layer norm, GELU with an 8-bit checkpoint, attention.

As in ``ops``: each function checks its arguments, allocates outputs and scratch through torch's
caching allocator and launches on the current stream of the tensors' device; nothing computes on
the CPU, and nothing here records gradients.

These calls are short on the GPU (a layer norm's training step of 8192 x 768 is 36 us of kernels), and in a
training step autograd runs the backward on a thread of its own, where every Python operation costs
two to three times what it does in a loop.  So they keep to few operations: the current stream and device
are read without building torch objects, arguments go to the library as plain values, and the library's
own checks are the only ones of what it checks.
"""
from __future__ import annotations

import ctypes
import struct

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


# The same, packed in one call: 4 int32, 7 int64, a double, 6 pointers, 12 strides, 4 pointers, 12 strides.
_ATTENTION = struct.Struct("@4i7qd6Q12q4Q12q")
assert _ATTENTION.size == ctypes.sizeof(AttentionArgs)


def bind(lib) -> None:
    """Signatures of ``lwl_layers.h`` on the loaded library."""
    i64, i32, sz, vp, dbl = ctypes.c_int64, ctypes.c_int, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_double
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
        "lwl_attention_check": (i32, [vp]),
        "lwl_attention_forward_workspace_size": (sz, [vp]),
        "lwl_attention_forward": (i32, [vp, vp, sz, vp]),
        "lwl_attention_backward_workspace_size": (sz, [vp]),
        "lwl_attention_backward": (i32, [vp, vp, sz, vp]),
    }
    for name, (res, args) in sigs.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args


_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _device_index(*tensors) -> int:
    """The GPU that all tensors (None: skipped) are on."""
    index = -1
    for t in tensors:
        if t is None:
            continue
        i = t.get_device()
        if i < 0 or (index >= 0 and i != index):
            N.require_cuda(*[t for t in tensors if t is not None])  # raises
        index = i
    return index


def _launch(index: int, fn, *args) -> None:
    """``fn(*args, stream)`` on the tensors' device and its current stream."""
    if index == _device():
        N.check(fn(*args, _stream(index)))
    else:
        with torch.cuda.device(index):
            N.check(fn(*args, _stream(index)))


def _ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _scratch(nbytes: int, like: torch.Tensor) -> torch.Tensor | None:
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes else None


def _dense(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


def _vector(name: str, t: torch.Tensor, n: int, dtype: torch.dtype) -> torch.Tensor:
    if t.shape != (n,) or t.dtype != dtype:
        raise N.BlockFHTArgumentError(f"{name} must be {n} values of {dtype}, got {tuple(t.shape)} of {t.dtype}")
    return _dense(t)


def _rows(what: str, x: torch.Tensor) -> tuple[int, int]:
    features = x.shape[-1] if x.dim() else 0
    if features == 0:
        raise N.BlockFHTArgumentError(f"{what} needs at least one feature, got {tuple(x.shape)}")
    return x.numel() // features, features


# ---------------------------------------------------------------- layer norm
def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, eps: float,
                       residual: torch.Tensor | None, keep_stats: bool):
    """``(out, sum, stats)`` over the last dimension of x; ``sum`` is None without a residual, ``stats``
    (float32 ``[2, rows]``: means, reciprocal deviations) unless ``keep_stats``."""
    index = _device_index(x, weight, bias, residual)
    rows, features = _rows("layer norm", x)
    weight = _vector("layer norm's weight", weight, features, weight.dtype)
    if bias is not None:
        bias = _vector("layer norm's bias", bias, features, weight.dtype)
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise N.BlockFHTArgumentError(
                f"residual must be {tuple(x.shape)} of {x.dtype}, got {tuple(residual.shape)} of {residual.dtype}")
        residual = _dense(residual)
    code, weight_code = N.dtype_code(x.dtype), N.dtype_code(weight.dtype)
    x = _dense(x)
    out = torch.empty_like(x)
    total = torch.empty_like(x) if residual is not None else None
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device) if keep_stats else None
    _launch(index, N.lib().lwl_layer_norm_forward, x.data_ptr(), _ptr(residual), weight.data_ptr(), _ptr(bias), code,
            weight_code, rows, features, eps, out.data_ptr(), _ptr(total), _ptr(stats))
    return out, total, stats


def layer_norm_backward(h: torch.Tensor, weight: torch.Tensor, stats: torch.Tensor, grad_out: torch.Tensor,
                        grad_sum: torch.Tensor | None, need_x: bool, need_weight: bool, need_bias: bool):
    """``(grad_x, grad_weight, grad_bias)``, None for what is not needed; ``h`` is what was normed (contiguous)."""
    index = _device_index(h, weight, stats, grad_out, grad_sum)
    rows, features = _rows("layer norm", h)
    dtype = h.dtype
    weight = _dense(weight)
    grad_out = _dense(grad_out if grad_out.dtype == dtype else grad_out.to(dtype))
    if grad_sum is not None:
        grad_sum = _dense(grad_sum if grad_sum.dtype == dtype else grad_sum.to(dtype))
    L = N.lib()
    gx = torch.empty_like(h) if need_x else None
    gw = torch.empty_like(weight) if need_weight else None
    gb = torch.empty_like(weight) if need_bias else None
    need = L.lwl_layer_norm_backward_workspace_size(rows, features) if need_weight or need_bias else 0
    ws = _scratch(need, h)
    _launch(index, L.lwl_layer_norm_backward, h.data_ptr(), weight.data_ptr(), stats.data_ptr(), grad_out.data_ptr(),
            _ptr(grad_sum), N.dtype_code(dtype), N.dtype_code(weight.dtype), rows, features, _ptr(gx), _ptr(gw), _ptr(gb),
            _ptr(ws), need)
    return gx, gw, gb


# ---------------------------------------------------------------- GELU, input kept in 8 bits
_FORMS = {"none": 0, "tanh": 1}


def _form(approximate: str) -> int:
    if approximate not in _FORMS:
        raise N.BlockFHTArgumentError(f"approximate must be 'none' or 'tanh', got {approximate!r}")
    return _FORMS[approximate]


def gelu8_forward(x: torch.Tensor, bias: torch.Tensor | None, approximate: str, keep: bool):
    """``(gelu(x + bias), codes, scales)`` over the last dimension of x; codes (int8 ``[rows, pitch]``) and
    scales (float32 ``[rows, groups]``) are None unless ``keep``."""
    index = _device_index(x, bias)
    rows, features = _rows("GELU checkpoint", x)
    code, form = N.dtype_code(x.dtype), _form(approximate)
    if bias is not None:
        bias = _vector("GELU's bias", bias, features, x.dtype)
    x = _dense(x)
    out = torch.empty_like(x)
    codes = scales = None
    if keep:
        codes = torch.empty((rows, (features + 7) // 8 * 8), dtype=torch.int8, device=x.device)
        scales = torch.empty((rows, -(-features // GELU8_GROUP)), dtype=torch.float32, device=x.device)
    _launch(index, N.lib().lwl_gelu8_forward, x.data_ptr(), _ptr(bias), code, form, rows, features, out.data_ptr(),
            _ptr(codes), _ptr(scales))
    return out, codes, scales


def gelu8_activation(codes: torch.Tensor, scales: torch.Tensor, shape: tuple[int, ...], dtype: torch.dtype,
                     approximate: str) -> torch.Tensor:
    """``gelu`` of what the checkpoint stands for, in ``shape`` and ``dtype``."""
    index = _device_index(codes, scales)
    out = torch.empty(shape, dtype=dtype, device=codes.device)
    _launch(index, N.lib().lwl_gelu8_activation, codes.data_ptr(), scales.data_ptr(), N.dtype_code(dtype),
            _form(approximate), codes.shape[0], shape[-1], out.data_ptr())
    return out


def gelu8_backward(codes: torch.Tensor, scales: torch.Tensor, grad_out: torch.Tensor, dtype: torch.dtype,
                   approximate: str, need_bias: bool):
    """``(grad_x, grad_bias)``; ``grad_out`` has the activation's shape."""
    index = _device_index(codes, scales, grad_out)
    grad_out = _dense(grad_out if grad_out.dtype == dtype else grad_out.to(dtype))
    rows, features = codes.shape[0], grad_out.shape[-1]
    L = N.lib()
    gx = torch.empty_like(grad_out)
    gb = torch.empty(features, dtype=dtype, device=gx.device) if need_bias else None
    need = L.lwl_gelu8_backward_workspace_size(rows, features) if need_bias else 0
    ws = _scratch(need, gx)
    _launch(index, L.lwl_gelu8_backward, codes.data_ptr(), scales.data_ptr(), grad_out.data_ptr(), N.dtype_code(dtype),
            _form(approximate), rows, features, gx.data_ptr(), _ptr(gb), _ptr(ws), need)
    return gx, gb


# ---------------------------------------------------------------- attention
ATTENTION_MAX_DIM = 128
_NO_GRADS = (0,) * 16


def _dense_dim(t: torch.Tensor) -> torch.Tensor:
    # the kernels take any strides but that of a head's values, which lie one after the other
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _attention_lengths(key_lengths: torch.Tensor | None, batch: int) -> torch.Tensor | None:
    if key_lengths is None or (key_lengths.dtype == torch.int32 and key_lengths.shape == (batch,)):
        return key_lengths if key_lengths is None else _dense(key_lengths)
    if key_lengths.shape != (batch,) or key_lengths.is_floating_point():
        raise N.BlockFHTArgumentError(f"attention: key_lengths must be {batch} integers, got {tuple(key_lengths.shape)} of "
                                      f"{key_lengths.dtype}")
    return _dense(key_lengths.to(torch.int32))


def _attention_shape(dtype, causal, scale, causal_offset, batch, heads, kv_heads, queries, keys, dim):
    """The arguments' fields up to the scale."""
    offset = 0 if causal_offset is None else int(causal_offset)
    if not -(1 << 62) < offset < 1 << 62:
        raise N.BlockFHTArgumentError(f"attention: causal_offset {offset} is too large")
    if scale is None:
        scale = dim ** -0.5 if dim else 0.0
    return (N.dtype_code(dtype), bool(causal), causal_offset is None, 0, offset, batch, heads, kv_heads, queries, keys, dim,
            float(scale))


def _attention_shape_of(q, k, v, causal, scale, causal_offset):
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise N.BlockFHTArgumentError(f"attention: q, k and v must be [batch, heads, tokens, head size], got "
                                      f"{tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    batch, heads, queries, dim = q.shape
    kb, kv_heads, keys, kd = shape = k.shape
    if shape != v.shape or kb != batch or kd != dim:
        raise N.BlockFHTArgumentError(f"attention: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not match")
    dtype = q.dtype
    if k.dtype != dtype or v.dtype != dtype:
        raise N.BlockFHTArgumentError(f"attention: q, k and v must have one type, got {dtype}, {k.dtype} and {v.dtype}")
    return _attention_shape(dtype, causal, scale, causal_offset, batch, heads, kv_heads, queries, keys, dim)


def _run_attention(index: int, like: torch.Tensor, forward: bool, *fields) -> None:
    L = N.lib()
    args = _ATTENTION.pack(*fields)
    need = (L.lwl_attention_forward_workspace_size if forward else L.lwl_attention_backward_workspace_size)(args)
    ws = _scratch(need, like)
    _launch(index, L.lwl_attention_forward if forward else L.lwl_attention_backward, args, _ptr(ws), need)


def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool, scale: float | None,
                      key_lengths: torch.Tensor | None, causal_offset: int | None, keep_lse: bool):
    """``(out, lse)`` for ``[batch, heads, tokens, head size]`` tensors; ``out`` lies in memory token by token
    (all heads of a token together); ``lse`` (float32 ``[batch, heads, queries]``) is None unless ``keep_lse``."""
    index = _device_index(q, k, v, key_lengths)
    shape = _attention_shape_of(q, k, v, causal, scale, causal_offset)
    batch, heads, queries, dim = q.shape
    lengths = _attention_lengths(key_lengths, batch)
    q, k, v = _dense_dim(q), _dense_dim(k), _dense_dim(v)
    out = torch.empty((batch, queries, heads, dim), dtype=q.dtype, device=q.device).transpose(1, 2)
    lse = torch.empty((batch, heads, queries), dtype=torch.float32, device=q.device) if keep_lse else None
    _run_attention(index, q, True, *shape, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(lse),
                   _ptr(lengths), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *out.stride()[:3], *_NO_GRADS)
    return out, lse


def attention_backward(q, k, v, out, lse, grad_out, causal, scale, key_lengths, causal_offset, grads) -> None:
    """Fills ``grads``, the three gradients like q, k and v (any strides, a head's values dense)."""
    index = _device_index(q, k, v, out, lse, grad_out, key_lengths)
    shape = _attention_shape_of(q, k, v, causal, scale, causal_offset)
    lengths = _attention_lengths(key_lengths, q.shape[0])
    q, k, v = _dense_dim(q), _dense_dim(k), _dense_dim(v)
    grad_out = _dense_dim(grad_out if grad_out.dtype == q.dtype else grad_out.to(q.dtype))
    gq, gk, gv = grads
    _run_attention(index, q, False, *shape, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
                   _ptr(lengths), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *out.stride()[:3],
                   grad_out.data_ptr(), gq.data_ptr(), gk.data_ptr(), gv.data_ptr(), *grad_out.stride()[:3],
                   *gq.stride()[:3], *gk.stride()[:3], *gv.stride()[:3])


def _packed(qkv: torch.Tensor, heads: int, kv_heads: int):
    """``(head size, strides, byte offsets of k and v)`` of a contiguous ``[batch, tokens, (heads + 2 kv_heads) *
    head size]``: the pieces by address, without a view of each."""
    tokens, width = qkv.shape[1], qkv.shape[2]
    dim = width // (heads + 2 * kv_heads)
    size = qkv.element_size()
    return dim, (tokens * width, dim, width), heads * dim * size, (heads + kv_heads) * dim * size


def attention_packed_forward(qkv: torch.Tensor, heads: int, kv_heads: int, causal: bool, scale: float | None,
                             key_lengths: torch.Tensor | None, causal_offset: int | None, keep_lse: bool):
    """``(out, lse)``; ``qkv`` contiguous, ``out`` ``[batch, tokens, heads * head size]``."""
    index = _device_index(qkv, key_lengths)
    dim, st, k_at, v_at = _packed(qkv, heads, kv_heads)
    batch, tokens = qkv.shape[0], qkv.shape[1]
    shape = _attention_shape(qkv.dtype, causal, scale, causal_offset, batch, heads, kv_heads, tokens, tokens, dim)
    lengths = _attention_lengths(key_lengths, batch)
    out = torch.empty((batch, tokens, heads * dim), dtype=qkv.dtype, device=qkv.device)
    lse = torch.empty((batch, heads, tokens), dtype=torch.float32, device=qkv.device) if keep_lse else None
    p = qkv.data_ptr()
    _run_attention(index, qkv, True, *shape, p, p + k_at, p + v_at, out.data_ptr(), _ptr(lse), _ptr(lengths), *st, *st, *st,
                   tokens * heads * dim, dim, heads * dim, *_NO_GRADS)
    return out, lse


def attention_packed_backward(qkv, out, lse, grad_out, heads, kv_heads, causal, scale, key_lengths, causal_offset):
    """The gradient of ``qkv``, in one tensor like it."""
    index = _device_index(qkv, out, lse, grad_out, key_lengths)
    dim, st, k_at, v_at = _packed(qkv, heads, kv_heads)
    batch, tokens = qkv.shape[0], qkv.shape[1]
    shape = _attention_shape(qkv.dtype, causal, scale, causal_offset, batch, heads, kv_heads, tokens, tokens, dim)
    lengths = _attention_lengths(key_lengths, batch)
    grad_out = _dense(grad_out if grad_out.dtype == qkv.dtype else grad_out.to(qkv.dtype))
    grad = torch.empty_like(qkv)
    p, g, ost = qkv.data_ptr(), grad.data_ptr(), (tokens * heads * dim, dim, heads * dim)
    _run_attention(index, qkv, False, *shape, p, p + k_at, p + v_at, out.data_ptr(), lse.data_ptr(), _ptr(lengths),
                   *st, *st, *st, *ost, grad_out.data_ptr(), g, g + k_at, g + v_at, *ost, *st, *st, *st)
    return grad


def once(backward):
    """A custom function's backward that cannot be differentiated itself.  What torch's
    ``once_differentiable`` guards against can only come about where the backward records a graph
    (``create_graph=True``); elsewhere its cost is spared."""
    guarded = torch.autograd.function.once_differentiable(backward)

    def call(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return call
