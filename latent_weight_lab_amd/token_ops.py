"""ctypes signatures of the C entries of ``include/lwl_tokens.h``: attention within a window and of a tree, tokens' log
probabilities.  Tensors reach them through the torch binding (``layer_ops``)."""
from __future__ import annotations

import ctypes

from .layer_ops import AttentionArgs


class LogProbsArgs(ctypes.Structure):
    """``lwl_log_probs_args``."""
    _fields_ = [("dtype", ctypes.c_int32), ("each", ctypes.c_int32), ("top", ctypes.c_int32), ("reserved", ctypes.c_int32),
                ("outer", ctypes.c_int64), ("inner", ctypes.c_int64), ("vocab", ctypes.c_int64),
                ("outer_stride", ctypes.c_int64), ("inner_stride", ctypes.c_int64), ("logits", ctypes.c_void_p),
                ("tokens", ctypes.c_void_p), ("log_probs", ctypes.c_void_p), ("entropy", ctypes.c_void_p),
                ("top_log_probs", ctypes.c_void_p), ("top_tokens", ctypes.c_void_p), ("stats", ctypes.c_void_p),
                ("grad_log_probs", ctypes.c_void_p), ("grad_entropy", ctypes.c_void_p), ("grad_top", ctypes.c_void_p),
                ("grad_logits", ctypes.c_void_p)]


def bind(lib) -> None:
    """Signatures of ``lwl_tokens.h`` on the loaded library."""
    i64, i32, sz, vp = ctypes.c_int64, ctypes.c_int, ctypes.c_size_t, ctypes.c_void_p
    attnp, logp = ctypes.POINTER(AttentionArgs), ctypes.POINTER(LogProbsArgs)
    sigs = {
        "lwl_attention_window_check": (i32, [attnp, i64, i64]),
        "lwl_attention_window_forward_workspace_size": (sz, [attnp, i64, i64]),
        "lwl_attention_window_forward": (i32, [attnp, i64, i64, vp, sz, vp]),
        "lwl_attention_window_backward_workspace_size": (sz, [attnp, i64, i64]),
        "lwl_attention_window_backward": (i32, [attnp, i64, i64, vp, sz, vp]),
        "lwl_attention_tree_check": (i32, [attnp]),
        "lwl_attention_tree_workspace_size": (sz, [attnp]),
        "lwl_attention_tree_forward": (i32, [attnp, vp, i64, vp, sz, vp]),
        "lwl_log_probs_check": (i32, [logp]),
        "lwl_log_probs_forward": (i32, [logp, vp]),
        "lwl_log_probs_backward": (i32, [logp, vp]),
    }
    for name, (res, args) in sigs.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
