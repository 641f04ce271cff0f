"""The layer operators' C entries and oracles without a GPU: structures, refusals, the formulas'
gradients against differences."""
from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

import layer_oracle as R
from latent_weight_lab_amd import _native as N
from latent_weight_lab_amd import attention, gelu_checkpoint8, layer_norm, layer_ops

ROOT = Path(__file__).resolve().parents[1]


def test_structures_match_the_header(tmp_path):
    fields = {"lwl_attention_args": layer_ops.AttentionArgs}
    lines = []
    for name, t in fields.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in t._fields_]
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include "lwl_layers.h"\nint main(void) {' + "\n".join(lines) + "return 0;}")
    subprocess.run(["gcc", f"-I{ROOT / 'include'}", str(src), "-o", str(tmp_path / "t")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for t in fields.values():
        want += [ctypes.sizeof(t)] + [getattr(t, f).offset for f, _ in t._fields_]
    assert got == want


def test_header_names_are_exported_and_bound():
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "lwl_layers.h").read_text(), flags=re.S)
    names = set(re.findall(r"\b(lwl_\w+)\(", text))
    assert len(names) == 15
    for n in names:
        assert getattr(N.lib(), n).argtypes is not None


@pytest.mark.parametrize("kw,rc", [({}, 0), ({"rows": 0}, 0), ({"rows": -1}, -1), ({"features": 0}, -1), ({"dtype": 3}, -2),
                                   ({"weight_dtype": 1}, -2), ({"eps": -1.0}, -1), ({"eps": float("inf")}, -1),
                                   ({"rows": 1 << 50}, -2), ({"features": 1 << 25}, -2)])
def test_norm_refusals(kw, rc):
    L = N.lib()
    a = {"dtype": 2, "weight_dtype": 0, "rows": 4, "features": 768, "eps": 1e-5, **kw}
    assert L.lwl_layer_norm_check(*a.values()) == rc
    if rc:
        assert L.lwl_last_error()
        assert L.lwl_layer_norm_forward(None, None, None, None, *a.values(), None, None, None, None) == rc


def test_null_pointers_and_workspaces_are_refused():
    # pointers of 256 are never dereferenced
    L = N.lib()
    shape = (2, 0, 100, 768)
    assert L.lwl_layer_norm_forward(None, None, None, None, *shape, 1e-5, None, None, None, None) == -1
    # a sum without a residual
    assert L.lwl_layer_norm_forward(256, None, 256, None, *shape, 1e-5, 256, 256, None, None) == -1
    # no stats
    assert L.lwl_layer_norm_backward(256, 256, None, 256, None, *shape, 256, 256, None, None, 0, None) == -1
    assert L.lwl_layer_norm_backward_workspace_size(100, 768) > 0
    assert L.lwl_layer_norm_backward(256, 256, 256, 256, None, *shape, 256, 256, None, None, 0, None) == -3
    assert L.lwl_gelu8_check(2, 5, 0) == -1 and L.lwl_gelu8_check(9, 5, 300) == -2 and L.lwl_gelu8_check(2, -1, 300) == -1
    assert L.lwl_gelu8_check(2, 5, 300) == 0 and L.lwl_gelu8_check(2, 1 << 50, 300) == -2
    assert L.lwl_gelu8_forward(None, None, 2, 0, 5, 300, None, None, None, None) == -1
    assert L.lwl_gelu8_activation(None, None, 2, 0, 5, 300, 256, None) == -1
    # codes off the 8-byte grid
    assert L.lwl_gelu8_forward(256, None, 2, 0, 5, 300, 256, 257, 256, None) == -1
    assert L.lwl_gelu8_backward(256, 256, None, 2, 0, 5, 300, None, None, None, 0, None) == -1
    assert L.lwl_gelu8_pitch(1) == 8 and L.lwl_gelu8_pitch(3072) == 3072
    assert L.lwl_attention_check(None) == -1
    t = attn_args()
    assert L.lwl_attention_forward(ctypes.byref(t), None, 0, None) == -1
    assert L.lwl_attention_backward(ctypes.byref(t), None, 0, None) == -1
    for f in ("q", "k", "v", "out", "lse", "grad_out", "grad_q", "grad_k", "grad_v"):
        setattr(t, f, 256)
    assert L.lwl_attention_backward_workspace_size(ctypes.byref(t)) >= 4 * 2 * 4 * 9
    assert L.lwl_attention_backward(ctypes.byref(t), None, 0, None) == -3


def attn_args(**kw):
    a = layer_ops.AttentionArgs()
    a.dtype, a.batch, a.heads, a.kv_heads, a.queries, a.keys, a.dim, a.scale = 2, 2, 4, 2, 9, 11, 64, 0.125
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,rc", [({}, 0), ({"dtype": 7}, -2), ({"heads": 3}, -1), ({"kv_heads": 0}, -1), ({"dim": 0}, -1),
                                   ({"dim": 129}, -2), ({"scale": 0.0}, -1), ({"scale": -1.0}, -1), ({"scale": 1e-60}, -1),
                                   ({"scale": float("nan")}, -1), ({"queries": -1}, -1), ({"keys": 1 << 31}, -2),
                                   ({"batch": 1 << 30, "heads": 4}, -2), ({"reserved": 1}, -1),
                                   ({"causal": 1, "causal_offset": 1 << 40}, -2), ({"keys": 0}, 0), ({"queries": 0}, 0)])
def test_attention_refusals(kw, rc):
    assert N.lib().lwl_attention_check(ctypes.byref(attn_args(**kw))) == rc


def test_cpu_tensors_are_refused():
    x = torch.randn(2, 4, 8, 16)
    for f in (lambda: attention(x, x, x), lambda: gelu_checkpoint8(x), lambda: layer_norm(x, x[0, 0, 0])):
        with pytest.raises(RuntimeError):
            f()


def central(f, x, d, eps=1e-6):
    return (f(x + eps * d) - f(x - eps * d)) / (2 * eps)


def test_formulas_match_differences():
    torch.manual_seed(0)
    r = lambda *s: torch.randn(*s, dtype=torch.float64)
    h, w, b, dy, d = r(3, 11), r(11), r(11), r(3, 11), r(3, 11)
    _, dx, dw, db = R.layer_norm(h, w, b, 1e-5, dy)
    f = lambda hh: (R.layer_norm(hh, w, b, 1e-5)[0] * dy).sum()
    assert abs(central(f, h, d) - (dx * d).sum()) < 1e-6
    dv = r(11)
    assert abs(central(lambda ww: (R.layer_norm(h, ww, b, 1e-5)[0] * dy).sum(), w, dv) - (dw * dv).sum()) < 1e-6
    assert abs(central(lambda bb: (R.layer_norm(h, w, bb, 1e-5)[0] * dy).sum(), b, dv) - (db * dv).sum()) < 1e-6
    q, k, v, do = r(2, 4, 5, 3), r(2, 2, 7, 3), r(2, 2, 7, 3), r(2, 4, 5, 3)
    ok = R.allowed(5, 7, [7, 4], 2, True, None)
    assert not ok[1, 0].any()  # an empty row
    g = R.attention(q, k, v, 0.7, ok, do)
    for i, name in enumerate(("dq", "dk", "dv")):
        t = (q, k, v)[i]
        step = r(*t.shape)
        f = lambda x: (R.attention(*[x if j == i else y for j, y in enumerate((q, k, v))], 0.7, ok)["o"] * do).sum()
        assert abs(central(f, t, step) - (g[name] * step).sum()) < 1e-6
    z = r(200) * 3
    for form in ("none", "tanh"):
        val, slope = R.gelu(z, form)
        assert torch.allclose(central(lambda x: R.gelu(x, form)[0], z, torch.ones_like(z)), slope, atol=1e-8)
        assert torch.allclose(val, torch.nn.functional.gelu(z, approximate=form), atol=1e-12)


def test_tiles_by_32_bit_offsets_only_where_they_reach(tmp_path):
    """A tile's rows are read at unsigned 32-bit byte offsets from its first, inside a range of (rows - 1) * stride +
    dim values: with descending rows offsets wrap, some of them into the range."""
    from latent_weight_lab_amd.build import hipcc

    strides = [s * m for s in (0, 8, 64, 120, 1 << 19, 1 << 23, (1 << 24) - 8, 1 << 24, 1 << 40, 1 << 57, 1 << 62)
               for m in (1, -1)]
    src = tmp_path / "t.cpp"
    src.write_text(f'''#include <cstdio>
#include "layer_launch.h"
int main() {{
  for (int64_t s : {{{", ".join(f"{s}LL" for s in strides)}}})
    for (int64_t size : {{2, 4}}) {{
      const int64_t stride[3] = {{0, 0, s}};
      std::printf("%lld %lld %d\\n", (long long)s, (long long)size, lwl::fast_rows((void*)256, stride, size));
    }}
}}''')
    rocm = Path(hipcc()).resolve().parents[1]
    subprocess.run([str(rocm / "llvm" / "bin" / "clang++"), "-std=c++17", "-D__HIP_PLATFORM_AMD__",
                    f"-I{ROOT / 'latent_weight_lab_amd' / 'csrc'}", f"-I{rocm / 'include'}", str(src), "-o",
                    str(tmp_path / "t")], check=True)
    out = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split()
    rows = [tuple(map(int, out[i:i + 3])) for i in range(0, len(out), 3)]
    assert len(rows) == 2 * len(strides)
    for stride, size, fast in rows:
        # every offset is the distance itself, and below the range that the hardware checks it against
        reach = [row * stride * size for row in range(64)]
        sound = all(0 <= r <= 63 * stride * size < 1 << 31 for r in reach)
        assert not fast or sound, (stride, size)
        if 0 <= stride <= 1 << 19:
            assert fast


@pytest.mark.parametrize("scale,rc", [(2.0 ** -100, 0), (2.0 ** 100, 0), (1e-39, -1), (3e38, -1), (float("inf"), -1)])
def test_scales_that_the_exponent_cannot_take_are_refused(scale, rc):
    """scale * log2(e) past float32's range gives 0 * infinity, its reciprocal past it log sums that are infinite."""
    assert N.lib().lwl_attention_check(ctypes.byref(attn_args(scale=scale))) == rc
