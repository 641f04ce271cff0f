"""The C entries of ``lwl_tokens.h`` and their oracles without a GPU: structures, refusals, the formulas' gradients against
differences."""
from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

import layer_oracle as R
import token_oracle as T
from latent_weight_lab_amd import _native as N
from latent_weight_lab_amd import attention, attention_tree, token_log_probs, token_ops
from test_layer_ops_cpu import attn_args, central

ROOT = Path(__file__).resolve().parents[1]


def test_structure_matches_the_header(tmp_path):
    t = token_ops.LogProbsArgs
    lines = ['printf("%zu\\n", sizeof(lwl_log_probs_args));']
    lines += [f'printf("%zu\\n", offsetof(lwl_log_probs_args, {f}));' for f, _ in t._fields_]
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include "lwl_tokens.h"\nint main(void) {' + "\n".join(lines) + "return 0;}")
    subprocess.run(["gcc", f"-I{ROOT / 'include'}", str(src), "-o", str(tmp_path / "t")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(t)] + [getattr(t, f).offset for f, _ in t._fields_]


def test_header_names_are_exported_and_bound():
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "lwl_tokens.h").read_text(), flags=re.S)
    names = set(re.findall(r"\b(lwl_\w+)\(", text))
    assert len(names) == 11
    for n in names:
        assert getattr(N.lib(), n).argtypes is not None


@pytest.mark.parametrize("kw,window,sinks,rc", [
    ({"causal": 1}, 1, 0, 0), ({"causal": 1}, 1 << 62, 1 << 62, 0), ({}, 5, 0, -1), ({"causal": 1}, 0, 0, -1),
    ({"causal": 1}, -1, 0, -1), ({"causal": 1}, 1, -1, -1), ({"causal": 1, "dim": 129}, 1, 0, -2),
    ({"causal": 1, "dtype": 9}, 1, 0, -2), ({"causal": 1, "queries": 0}, 3, 1, 0)])
def test_window_refusals(kw, window, sinks, rc):
    L = N.lib()
    a = ctypes.byref(attn_args(**kw))
    assert L.lwl_attention_window_check(a, window, sinks) == rc
    if rc:
        assert L.lwl_last_error()
        assert L.lwl_attention_window_forward(a, window, sinks, None, 0, None) == rc
        assert L.lwl_attention_window_backward(a, window, sinks, None, 0, None) == rc
        assert L.lwl_attention_window_forward_workspace_size(a, window, sinks) == 0


@pytest.mark.parametrize("kw,rc", [({}, 0), ({"causal": 1}, -1), ({"bottom_right": 1}, -1), ({"causal_offset": 3}, -1),
                                   ({"queries": 128}, 0), ({"queries": 129}, -2),
                                   ({"batch": 1, "queries": 128, "heads": 1 << 27, "kv_heads": 1, "keys": 1}, -2), ({"heads": 3}, -1), ({"keys": 0}, 0)])
def test_tree_refusals(kw, rc):
    L = N.lib()
    a = ctypes.byref(attn_args(**kw))
    assert L.lwl_attention_tree_check(a) == rc
    if rc:
        assert L.lwl_last_error()
        assert L.lwl_attention_tree_forward(a, 256, 0, None, 0, None) == rc


def log_args(**kw):
    a = token_ops.LogProbsArgs()
    a.dtype, a.each, a.top, a.outer, a.inner, a.vocab, a.outer_stride, a.inner_stride = 2, 1, 0, 1, 5, 100, 0, 100
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,rc", [({}, 0), ({"dtype": 5}, -2), ({"reserved": 1}, -1), ({"outer": -1}, -1), ({"vocab": 0}, -1),
                                   ({"each": -1}, -1), ({"each": 65}, -2), ({"top": 101}, -1), ({"top": 65}, -2),
                                   ({"top": 64}, 0), ({"vocab": (1 << 30) + 1}, -2), ({"outer": 1 << 30, "inner": 2}, -2),
                                   ({"outer": 1 << 40, "inner": 1 << 40}, -2), ({"inner": 0}, 0)])
def test_log_probs_refusals(kw, rc):
    L = N.lib()
    a = ctypes.byref(log_args(**kw))
    assert L.lwl_log_probs_check(a) == rc
    if rc:
        assert L.lwl_last_error()
        assert L.lwl_log_probs_forward(a, None) == rc and L.lwl_log_probs_backward(a, None) == rc


def test_null_pointers_and_workspaces_are_refused():
    # pointers of 256 are never dereferenced
    L = N.lib()
    t = attn_args(causal=1, queries=300, keys=4000)
    assert L.lwl_attention_window_forward(ctypes.byref(t), 5, 0, None, 0, None) == -1
    assert L.lwl_attention_window_backward(ctypes.byref(t), 5, 0, None, 0, None) == -1
    for f in ("q", "k", "v", "out", "lse", "grad_out", "grad_q", "grad_k", "grad_v"):
        setattr(t, f, 256)
    assert L.lwl_attention_window_backward(ctypes.byref(t), 5, 0, None, 0, None) == -3
    t = attn_args(queries=20, keys=100_000)
    t.q = t.k = t.v = t.out = 256
    assert L.lwl_attention_tree_forward(ctypes.byref(t), None, 0, None, 0, None) == -1
    assert L.lwl_attention_tree_workspace_size(ctypes.byref(t)) > 0
    assert L.lwl_attention_tree_forward(ctypes.byref(t), 256, 0, None, 0, None) == -3
    assert L.lwl_attention_tree_check(None) == -1 and L.lwl_log_probs_check(None) == -1
    assert L.lwl_attention_window_check(None, 1, 0) == -1
    a = log_args()
    assert L.lwl_log_probs_forward(ctypes.byref(a), None) == -1
    a.logits = 256
    for kw in ({}, {"tokens": 256}, {"log_probs": 256}, {"tokens": 256, "log_probs": 256, "top": 2},
               {"tokens": 256, "log_probs": 256, "top_tokens": 256}):
        assert L.lwl_log_probs_forward(ctypes.byref(log_args(logits=256, **kw)), None) == -1
    for kw in ({}, {"stats": 256}, {"stats": 256, "grad_logits": 256, "grad_log_probs": 256},
               {"stats": 256, "grad_logits": 256, "grad_entropy": 256}, {"stats": 256, "grad_logits": 256, "grad_top": 256}):
        assert L.lwl_log_probs_backward(ctypes.byref(log_args(logits=256, **kw)), None) == -1


@pytest.mark.parametrize("kw", [{"batch": 0, "keys": 100_000}, {"batch": 0, "keys": 100_000, "queries": 40},
                                {"batch": 0, "keys": 0, "queries": 0}, {"keys": 0}, {"queries": 0, "keys": 100_000}])
def test_workspaces_of_empty_calls(kw):
    L = N.lib()
    for lengths in (None, 256):
        a = attn_args(**kw)
        a.key_lengths = lengths
        assert L.lwl_attention_tree_workspace_size(ctypes.byref(a)) < 1 << 31
        a.causal = 1
        assert L.lwl_attention_window_forward_workspace_size(ctypes.byref(a), 100, 4) < 1 << 31
        assert L.lwl_attention_window_backward_workspace_size(ctypes.byref(a), 100, 4) < 1 << 31


def test_workspaces_grow_with_the_window_only():
    """A long sequence's ranges are those of its window, and sinks' blocks have their own."""
    L = N.lib()
    a = attn_args(causal=1, batch=1, heads=2, kv_heads=2, queries=1, keys=1 << 20)
    near, far = (L.lwl_attention_window_forward_workspace_size(ctypes.byref(a), w, 0) for w in (1024, 1 << 20))
    assert 0 < near < far
    a = attn_args(causal=1, batch=1, heads=2, kv_heads=2, queries=1 << 15, keys=1 << 15)
    no, some = (L.lwl_attention_window_backward_workspace_size(ctypes.byref(a), 256, s) for s in (0, 4))
    assert no < some


def test_cpu_tensors_are_refused():
    x = torch.randn(2, 4, 8, 16)
    p = torch.zeros(8, dtype=torch.int32)
    for f in (lambda: attention(x, x, x, causal=True, window=3), lambda: attention_tree(x, x, x, p),
              lambda: token_log_probs(x, torch.zeros(2, 4, 8, dtype=torch.long))):
        with pytest.raises(RuntimeError):
            f()


def test_which_pairs_are_allowed():
    ok = T.window_allowed(4, 6, None, 1, None, 2, 1)[0].int().tolist()
    assert ok == [[1, 1, 1, 0, 0, 0], [1, 0, 1, 1, 0, 0], [1, 0, 0, 1, 1, 0], [1, 0, 0, 0, 1, 1]]
    ok = T.window_allowed(2, 6, [3], 1, 3, 2, 0)[0].int().tolist()  # positions 3 and 4 of a sequence of 3 keys
    assert ok == [[0, 0, 1, 0, 0, 0], [0, 0, 0, 0, 0, 0]]
    ok = T.tree_allowed([[-1, 0, 0, 2, 7]], 7, [6], 1)[0].int().tolist()
    assert ok == [[1, 1, 0, 0, 0, 0, 0], [1, 1, 1, 0, 0, 0, 0], [1, 1, 0, 1, 0, 0, 0], [1, 1, 0, 1, 1, 0, 0],
                  [1, 0, 0, 0, 0, 1, 0]]


def test_formulas_match_differences():
    torch.manual_seed(0)
    r = lambda *s: torch.randn(*s, dtype=torch.float64)
    z, tokens = r(3, 19), torch.tensor([[3, 3], [-1, 18], [0, 40]])
    g, gh, gtop, step = r(3, 2), r(3), r(3, 4), r(3, 19)
    res = T.log_probs(z, tokens, g, gh, gtop, 4)

    def f(x):
        v = T.log_probs(x, tokens, top=4)
        return (torch.nan_to_num(v["log_probs"]) * g).sum() + (v["entropy"] * gh).sum() + (v["top_log_probs"] * gtop).sum()

    assert abs(central(f, z, step) - (res["grad"] * step).sum()) < 1e-6
    q, k, v, do = r(2, 4, 5, 3), r(2, 2, 9, 3), r(2, 2, 9, 3), r(2, 4, 5, 3)
    ok = T.window_allowed(5, 9, [9, 4], 2, None, 3, 1)
    grads = R.attention(q, k, v, 0.7, ok, do)
    for i, name in enumerate(("dq", "dk", "dv")):
        x = (q, k, v)[i]
        step = r(*x.shape)
        f = lambda y: (R.attention(*[y if j == i else t for j, t in enumerate((q, k, v))], 0.7, ok)["o"] * do).sum()
        assert abs(central(f, x, step) - (grads[name] * step).sum()) < 1e-6
