"""Calls that would take more workgroups than a launch has are refused before it, by the C entries."""
from __future__ import annotations

import ctypes

import pytest

from latent_weight_lab_amd import _native as N
from test_layer_ops_cpu import attn_args
from test_token_ops_cpu import log_args

MOST = ((1 << 32) - 1) // 256  # workgroups of 256 threads


def filled(**kw):
    a = attn_args(**kw)
    for f in ("q", "k", "v", "out", "lse", "grad_out", "grad_q", "grad_k", "grad_v"):
        setattr(a, f, 256)  # never dereferenced
    return a


@pytest.mark.parametrize("kw", [
    {"batch": MOST + 1, "heads": 1, "kv_heads": 1, "queries": 1, "keys": 1},            # a token each
    {"batch": MOST // 2 + 1, "heads": 2, "kv_heads": 2, "queries": 17, "keys": 1},      # rows
    {"batch": (MOST + 1) // 4, "heads": 8, "kv_heads": 8, "queries": 64, "keys": 64}])
def test_attention(kw):
    L = N.lib()
    assert L.lwl_attention_tree_check(ctypes.byref(attn_args(**kw))) == -2
    a = ctypes.byref(filled(**kw))
    assert L.lwl_attention_tree_forward(a, 256, 0, 256, 1 << 62, None) == -2
    assert b"workgroups" in L.lwl_last_error()
    assert L.lwl_attention_tree_workspace_size(a) == 0
    a = ctypes.byref(filled(causal=1, **kw))
    for call in (lambda: L.lwl_attention_forward(a, 256, 1 << 62, None),
                 lambda: L.lwl_attention_window_forward(a, 3, 1, 256, 1 << 62, None),
                 lambda: L.lwl_attention_backward(a, 256, 1 << 62, None),
                 lambda: L.lwl_attention_window_backward(a, 3, 1, 256, 1 << 62, None)):
        assert call() == -2
        assert b"workgroups" in L.lwl_last_error()


def test_attention_whose_backward_alone_is_past_it():
    """Few queries over many keys: a forward pass that fits, key blocks that do not."""
    L = N.lib()
    a = filled(batch=1 << 16, heads=16, kv_heads=4, queries=4, keys=128 * 70, causal=1)
    assert L.lwl_attention_check(ctypes.byref(a)) == 0
    assert L.lwl_attention_backward(ctypes.byref(a), 256, 1 << 62, None) == -2
    assert L.lwl_attention_window_backward(ctypes.byref(a), 3, 1, 256, 1 << 62, None) == -2


@pytest.mark.parametrize("kw", [{"batch": MOST, "heads": 1, "kv_heads": 1, "queries": 1, "keys": 1},
                                {"batch": MOST, "heads": 16, "kv_heads": 1, "queries": 1, "keys": 1},
                                {"batch": MOST // 2, "heads": 2, "kv_heads": 2, "queries": 17, "keys": 1}])
def test_what_fits_is_taken(kw):
    L = N.lib()
    assert L.lwl_attention_tree_check(ctypes.byref(attn_args(**kw))) == 0
    assert L.lwl_attention_check(ctypes.byref(attn_args(causal=1, **kw))) == 0
    assert L.lwl_attention_window_check(ctypes.byref(attn_args(causal=1, **kw)), 3, 1) == 0


@pytest.mark.parametrize("kw,rc", [({"inner": MOST + 1, "vocab": 3}, 0), ({"inner": (1 << 31) - 1, "vocab": 3}, 0),
                                   ({"inner": 1 << 31, "vocab": 3}, -2), ({"outer": 1 << 20, "inner": 1 << 10, "vocab": 50_000}, -2)])
def test_log_probs(kw, rc):
    """Rows go on in a grid's second axis, up to 2^31 rows and parts of rows."""
    assert N.lib().lwl_log_probs_check(ctypes.byref(log_args(**kw))) == rc
