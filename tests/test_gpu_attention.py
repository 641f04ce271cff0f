"""Attention (``attention``, ``attention_packed``, ``lwl_attention_*``) against float64, both directions.

Bounds, elementwise (``layer_oracle.attention`` gives the sizes): a probability is off by gamma (the score's
float32 error) and, where it is an operand of a 16-bit product, by u; a gradient of a score by twice that
and by u again for its own rounding and for the rounded output inside D.  With T the sum of the sizes of a
result's terms: |error| <= (2 u + gamma) T + u |result| forward, (4 u + 4 gamma) T + u |result| backward.
"""
from __future__ import annotations

import ctypes

import pytest
import torch

import layer_oracle as R
from conftest import gpu_available
from latent_weight_lab_amd import _native as N
from latent_weight_lab_amd import attention, attention_packed, layer_ops

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def make(b, h, hk, tq, tk, d, dt, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dt)
    return r(b, tq, h, d).transpose(1, 2), r(b, tk, hk, d).transpose(1, 2), r(b, tk, hk, d).transpose(1, 2), \
        r(b, tq, h, d).transpose(1, 2)


def compare(got, res, name, dt, factor, gamma):
    u = R.U[dt]
    want, terms = res[name], res[name + "_terms"]
    err = (got.double().cpu() - want).abs()
    bound = (factor * u + (factor - 1) * gamma) * terms + u * want.abs() + R.TINY[dt]
    assert torch.isfinite(got).all(), name
    assert (err <= bound).all(), (name, (err / bound).max().item())


def run(q, k, v, do, dt, causal=False, lengths=None, offset=None, scale=None, step=True):
    b, h, tq, d = q.shape
    tk = k.shape[2]
    sc = scale or d ** -0.5
    ok = R.allowed(tq, tk, lengths, b, causal, offset)
    res = R.attention(q, k, v, sc, ok, do if step else None)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    gq, gk, gv = (t.cuda() for t in (q, k, v))
    out, lse = layer_ops.attention_forward(gq, gk, gv, causal, scale, lens, offset, True)
    compare(out, res, "o", dt, 2, res["gamma"])
    some = ok.any(2).unsqueeze(1).expand(-1, h, -1)
    assert (lse.cpu()[~some] == float("-inf")).all()
    if some.any():
        off = (lse.double().cpu() - res["lse"]).abs()[some]
        assert (off <= res["gamma"].squeeze(-1)[some] + 2.0 ** -20 * (1 + res["lse"].abs()[some])).all()
    if step:
        gq, gk, gv = (t.requires_grad_() for t in (gq, gk, gv))
        o = attention(gq, gk, gv, causal=causal, scale=scale, key_lengths=lens, causal_offset=offset)
        assert torch.equal(o, out)
        for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(o, (gq, gk, gv), do.cuda())):
            compare(g, res, name, dt, 4, res["gamma_all"])


# batch, heads, key heads, queries, keys, head size: one of everything, a tile's last and one more, several
# workgroups, more queries than keys, few queries over many keys (ranges of keys joined), shared key heads
SHAPES = [(1, 1, 1, 1, 1, 1), (2, 3, 3, 1, 1, 64), (1, 2, 2, 5, 3, 7), (2, 2, 1, 32, 64, 32), (1, 2, 2, 33, 65, 33),
          (2, 4, 2, 64, 64, 64), (1, 3, 1, 127, 129, 64), (1, 2, 2, 129, 127, 96), (2, 2, 2, 200, 333, 80),
          (1, 4, 2, 300, 300, 128), (1, 2, 1, 130, 1000, 65), (1, 6, 2, 257, 70, 100), (3, 4, 4, 3, 700, 64),
          (1, 8, 1, 2, 1300, 128), (1, 20, 1, 1, 900, 48), (1, 1, 1, 17, 2100, 64), (2, 1, 1, 700, 31, 24)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("causal", [False, True])
def test_step_matches_float64(shape, dtype, causal):
    b, h, hk, tq, tk, d = shape
    q, k, v, do = make(*shape, DT[dtype], sum(shape))
    run(q, k, v, do, DT[dtype], causal=causal)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("tq,tk,lengths", [(40, 150, [0, 1, 150, 63, 64, 65]), (200, 200, [200, 0, 5, 128, 129, 199]),
                                           (1, 400, [1, 0, 400, 31, 32, 33]), (4, 1200, [3, 1200, 0, 257, 1, 800])])
@pytest.mark.parametrize("causal,offset", [(False, None), (True, None), (True, 0), (True, -3), (True, 100)])
def test_lengths_and_offsets(dtype, tq, tk, lengths, causal, offset):
    """Empty and short sequences, with anything at all past their ends."""
    q, k, v, do = make(6, 4, 2, tq, tk, 64, DT[dtype], tq + tk)
    k, v = k.clone(), v.clone()
    for i, n in enumerate(lengths):
        k[i, :, n:] = float("nan")
        v[i, :, n:] = float("inf")
    # queries that see nothing may hold anything too
    ok = R.allowed(tq, tk, lengths, 6, causal, offset)
    q, do = q.clone(), do.clone()
    none = ~ok.any(2)
    q.permute(0, 2, 1, 3)[none] = float("nan")
    do.permute(0, 2, 1, 3)[none] = float("inf")
    run(q, k, v, do, DT[dtype], causal=causal, lengths=lengths, offset=offset)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_layouts(dtype):
    """Strides of every kind give what contiguous tensors give, bit for bit."""
    dt = DT[dtype]
    q, k, v, do = (t.cuda() for t in make(2, 4, 2, 70, 90, 72, dt, 5))
    want = attention(q.contiguous(), k.contiguous(), v.contiguous(), causal=True)

    def odd(t):  # odd offset and odd strides
        b, h, n, d = t.shape
        buf = torch.full((b, n, h, d + 5), float("nan"), dtype=dt, device="cuda")
        view = buf[..., 3:3 + d].transpose(1, 2)
        view.copy_(t)
        return view

    def columns(t):  # a head's values apart
        return t.transpose(2, 3).contiguous().transpose(2, 3)

    for make_view in (lambda t: t, odd, columns):
        leaves = [make_view(t).detach().requires_grad_() for t in (q, k, v)]
        o = attention(*leaves, causal=True)
        assert torch.equal(o, want)
        assert o.transpose(1, 2).is_contiguous()
        grads = torch.autograd.grad(o, leaves, make_view(do))
        if make_view is odd:
            assert all(torch.equal(a, b) for a, b in zip(grads, first))
        first = grads
    # one key head shared by stride 0, its gradient summed by autograd
    k1, v1 = (t[:, :1].detach().requires_grad_() for t in (k, v))
    o = attention(q, k1.expand(-1, 4, -1, -1), v1.expand(-1, 4, -1, -1))
    assert torch.equal(o, attention(q, k1, v1))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("heads,kv_heads,dim,t", [(4, 4, 64, 100), (6, 2, 40, 77), (3, 1, 9, 33)])
def test_packed_is_the_same(dtype, heads, kv_heads, dim, t):
    dt = DT[dtype]
    g = torch.Generator().manual_seed(t)
    x = torch.randn(2, t, (heads + 2 * kv_heads) * dim, generator=g).to(dt).cuda().requires_grad_()
    dy = torch.randn(2, t, heads * dim, generator=g).to(dt).cuda()
    y = attention_packed(x, heads, kv_heads)
    (gx,) = torch.autograd.grad(y, x, dy)
    q, k, v = (s.unflatten(-1, (-1, dim)).transpose(1, 2)
               for s in x.split([heads * dim, kv_heads * dim, kv_heads * dim], -1))
    o = attention(q, k, v, causal=True).transpose(1, 2).reshape(2, t, -1)
    assert torch.equal(y, o)
    assert torch.equal(gx, torch.autograd.grad(o, x, dy)[0])


def test_tokens_over_a_cache_equal_the_prompt():
    """One to five tokens at a time over a preallocated cache give the rows of the whole prompt's pass."""
    q, k, v, _ = (t.cuda() for t in make(2, 6, 3, 200, 200, 64, torch.float32, 9))
    whole = attention(q, k, v, causal=True)
    cache_k, cache_v = (torch.full((2, 512, 3, 64), float("nan"), device="cuda") for _ in range(2))
    done = 0
    for n in [100, 1, 5, 1, 2, 60, 31]:
        cache_k[:, done:done + n] = k[:, :, done:done + n].transpose(1, 2)
        cache_v[:, done:done + n] = v[:, :, done:done + n].transpose(1, 2)
        lens = torch.full((2,), done + n, device="cuda")
        o = attention(q[:, :, done:done + n], cache_k.transpose(1, 2), cache_v.transpose(1, 2), causal=True, key_lengths=lens)
        assert (o - whole[:, :, done:done + n]).abs().max() < 1e-5
        o = attention(q[:, :, done:done + n], cache_k[:, :done + n].transpose(1, 2), cache_v[:, :done + n].transpose(1, 2),
                      causal=True)
        assert (o - whole[:, :, done:done + n]).abs().max() < 1e-5
        done += n


def test_offsets_past_32_bits():
    """A cache whose tokens lie more than 2^31 values apart."""
    stride = (1 << 31) // 300 + 64
    buf = torch.zeros(stride * 400, dtype=torch.float16, device="cuda")
    q, k, v, _ = (t.cuda() for t in make(1, 1, 1, 200, 400, 64, torch.float16, 2))
    bk = buf.as_strided((1, 1, 400, 64), (0, 0, stride, 1))
    bv = buf[128:].as_strided((1, 1, 400, 64), (0, 0, stride, 1))
    bk.copy_(k)
    bv.copy_(v)
    for n in (200, 1):
        assert torch.equal(attention(q[:, :, :n], bk, bv), attention(q[:, :, :n], k, v))


def test_extreme_scores():
    for dt in DT.values():
        q = torch.zeros(1, 1, 40, 64, dtype=dt)
        k = torch.zeros(1, 1, 300, 64, dtype=dt)
        v = torch.randn(1, 1, 300, 64, generator=torch.Generator().manual_seed(1)).to(dt)
        q[..., 0] = 100.0
        k[0, 0, :, 0] = torch.linspace(-200.0, 200.0, 300).to(dt)  # scores of -2500 .. 2500, rising and then falling
        for kk in (k, k.flip(2)):
            run(q, kk, v, v[:, :, :40].clone(), dt)
        q[0, 0, 3, 0] = float("nan")
        o = attention(q.cuda(), k.cuda(), v.cuda())
        assert o[0, 0, 3].isnan().all() and torch.isfinite(o[0, 0, :3]).all() and torch.isfinite(o[0, 0, 4:]).all()


def test_repeats_streams_and_graph():
    q, k, v, do = (t.cuda() for t in make(2, 6, 2, 300, 300, 64, torch.bfloat16, 8))
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]

    def step():
        o = attention(*leaves, causal=True)
        return [o, *torch.autograd.grad(o, leaves, do)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    # a decoding step in a graph: the lengths are read on the device
    ck, cv = (torch.randn(2, 2000, 2, 64, device="cuda").bfloat16().transpose(1, 2) for _ in range(2))
    lens = torch.tensor([5, 7], dtype=torch.int32, device="cuda")
    q1 = q[:, :, :1].contiguous()
    graph = torch.cuda.CUDAGraph()
    attention(q1, ck, cv, causal=True, key_lengths=lens)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        o = attention(q1, ck, cv, causal=True, key_lengths=lens)
    for n in (5, 2000, 900, 1):
        lens.fill_(n)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, attention(q1, ck, cv, causal=True, key_lengths=lens))


def test_refusals():
    q = torch.randn(2, 4, 8, 32, device="cuda")
    k = torch.randn(2, 2, 9, 32, device="cuda")
    lens = torch.tensor([3, 4], device="cuda")
    attention(q, k, k, key_lengths=lens)
    for bad in (lambda: attention(q, k, k[:, :, :8]), lambda: attention(q, k[:1], k[:1]), lambda: attention(q, k.half(), k),
                lambda: attention(q[:, :3], k, k), lambda: attention(q[0], k, k), lambda: attention(q, k, k, scale=0.0),
                lambda: attention(q, k, k, scale=-1.0), lambda: attention(q, k, k, scale=float("nan")),
                lambda: attention(q, k, k, key_lengths=lens[:1]), lambda: attention(q, k, k, key_lengths=lens.float()),
                lambda: attention(q.cpu(), k.cpu(), k.cpu()), lambda: attention(q.double(), k.double(), k.double()),
                lambda: attention(q.repeat(1, 1, 1, 5), k.repeat(1, 1, 1, 5), k.repeat(1, 1, 1, 5)),
                lambda: attention(q, k, k, key_lengths=lens.cpu()), lambda: attention_packed(q[0], 3),
                lambda: attention(q, k, k, causal=True, causal_offset=1 << 40)):
        with pytest.raises((RuntimeError, ValueError)):
            bad()


@pytest.mark.parametrize("tq,tk,b", [(0, 5, 2), (3, 0, 2), (0, 0, 1), (4, 6, 0)])
def test_empty_tensors(tq, tk, b):
    q = torch.randn(b, 4, tq, 32, device="cuda", requires_grad=True)
    k = torch.randn(b, 2, tk, 32, device="cuda", requires_grad=True)
    v = torch.randn(b, 2, tk, 32, device="cuda", requires_grad=True)
    o = attention(q, k, v)
    assert o.shape == q.shape and (o == 0).all()
    for g, t in zip(torch.autograd.grad(o.sum(), (q, k, v)), (q, k, v)):
        assert g.shape == t.shape and (g == 0).all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(2, 2, 1, 70, 130, 7), (1, 2, 2, 33, 65, 21), (1, 2, 1, 140, 200, 69),
                                   (2, 2, 2, 66, 64, 102), (2, 4, 2, 1, 150, 43), (1, 2, 1, 3, 70, 86)])
@pytest.mark.parametrize("gap", [1, 9])
def test_nothing_beside_a_row_counts(dtype, shape, gap):
    """Head sizes that fill no eight values, in rows `gap` values apart that hold NaN, as does all around the
    tensor: the results are those of the tensors alone."""
    b, h, hk, tq, tk, d = shape
    clean = [t.cuda() for t in make(*shape, DT[dtype], 5)]

    def hidden(t):
        room = torch.full((t.shape[0], t.shape[1] + 2, t.shape[2] + 2, d + gap), float("nan"), dtype=t.dtype, device="cuda")
        view = room[:, 1:-1, 1:-1, :d]
        view.copy_(t)
        return view

    def step(q, k, v, do):
        out, lse = layer_ops.attention_forward(q, k, v, True, None, None, None, True)
        return out, *layer_ops.attention_backward(q, k, v, out, lse, do, True, None, None, None)

    for want, got in zip(step(*clean), step(*map(hidden, clean))):
        assert torch.isfinite(got).all() and torch.equal(want, got)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(1, 2, 1, 40, 1500, 32), (2, 3, 1, 65, 1030, 64), (1, 1, 1, 129, 2100, 100)])
@pytest.mark.parametrize("lengths,causal", [(False, True), (True, True), (True, False)])
def test_few_queries_over_many_keys(dtype, shape, lengths, causal):
    """Both passes of the backward in ranges, of which some hold no key."""
    b, h, hk, tq, tk, d = shape
    q, k, v, do = make(*shape, DT[dtype], sum(shape))
    run(q, k, v, do, DT[dtype], causal=causal, lengths=[tk // 3, 0][:b] if lengths else None)


@pytest.mark.parametrize("std", [1.0, 1e-3, 1e-4])
@pytest.mark.parametrize("shape", [(1, 4, 1, 2048, 4096, 64), (1, 2, 2, 1100, 3000, 128), (1, 2, 2, 1500, 2000, 80)])
def test_float16_gradients_of_small_dout(shape, std):
    """Long rows times small gradients, where probability times gradient is below float16's normal range.

    In the L2 norm the gradients are off by their own rounding, which is what the exact ones rounded are off by, and by
    the relative error of their terms: a rounding (2^-11) each of P or dS, of out inside D and of the product's
    start, doubled for the float32 steps between."""
    q, k, v, do = make(*shape, torch.float16, 3)
    do = (do.float() * std).half()
    d = shape[-1]
    res = R.attention(q, k, v, d ** -0.5, torch.ones(1, *shape[3:5], dtype=torch.bool), do)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(attention(*leaves), leaves, do.cuda())):
        want = res[name]
        off, least = (g.double().cpu() - want).norm(), (want.half().double() - want).norm()
        assert off <= least + 6 * R.U[torch.float16] * want.norm(), (name, (off / want.norm()).item())


def test_float16_gradients_of_large_dout():
    """Gradients of scores past float16's range, of which those of q, k and v are well inside."""
    q, k, v, do = make(1, 2, 1, 200, 3, 64, torch.float16, 3)
    q, k, v, do = (0.05 * q).half(), (0.05 * k).half(), (4 * v).half(), (1000 * do).half()
    do[:, :, 100:] *= 4  # later tiles larger: the sums are rescaled
    ds = (do.double() @ v.double().transpose(2, 3).repeat_interleave(2, 1)) / 3
    assert ds.abs().max() > 65504
    run(q, k, v, do, torch.float16)


def test_float16_gradients_of_large_values():
    """Values whose rows are longer than float16's range, upstream gradients along them: the scores' gradients over
    the length of dout's row leave it too, and dQ does not."""
    q, k, _, _ = make(1, 1, 1, 70, 2, 64, torch.float16, 4)
    v = (20000 * torch.sign(make(1, 1, 1, 2, 2, 64, torch.float16, 5)[1])).half()
    v[:, :, 1] = -v[:, :, 0]
    do = (1e-6 * v[:, :, :1]).expand(-1, -1, 70, -1).clone()
    for tk in (2, 130):  # the second: in a later tile, beside small ones
        kk, vv = torch.zeros(1, 1, tk, 64).half(), torch.zeros(1, 1, tk, 64).half()
        kk[:, :, -2:], vv[:, :, -2:] = k, v
        vv[:, :, :-2] = 1.0
        run(q, kk, vv, do, torch.float16, scale=0.01)


def test_what_does_not_fit_the_forward_is_refused():
    q, k, v, do = (t.cuda() for t in make(2, 4, 2, 9, 12, 32, torch.float16, 1))
    out, lse = layer_ops.attention_forward(q, k, v, False, None, None, None, True)
    back = lambda out, lse, do: layer_ops.attention_backward(q, k, v, out, lse, do, False, None, None, None)
    back(out, lse, do)
    back(out, lse, do.float())  # converted
    for args in [(out, lse.half(), do), (out, lse.double(), do), (out, lse.view(-1), do), (out, lse[:, :2], do),
                 (out, lse.transpose(0, 1), do), (out, torch.cat([lse, lse], 2)[:, :, ::2], do), (out.float(), lse, do),
                 (out.bfloat16(), lse, do), (out[:, :, :8], lse, do), (out, lse, do[:1]), (out, lse.cpu(), do)]:
        with pytest.raises(RuntimeError):
            back(*args)


def test_saved_tensors_in_another_layout_or_type():
    """A caller's hooks may give saved tensors back in another layout, not in another type."""
    x = torch.randn(2, 20, 3 * 64, device="cuda", requires_grad=True)
    y = attention_packed(x, 2)
    want = torch.autograd.grad(y.sum(), x)[0]
    apart = lambda t: torch.stack([t, t], -1)[..., 0] if t.is_floating_point() else t
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: apart(t) if t.shape[-1] != 20 else t):
        y = attention_packed(x, 2)
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], want)
    for change in (apart, torch.Tensor.half):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: change(t) if t.shape[-1] == 20 else t):
            y = attention_packed(x, 2)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y.sum(), x)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("tq,tk,d", [(1, 300, 64), (70, 150, 64), (70, 150, 61)])
def test_rows_in_descending_order(dtype, tq, tk, d):
    """Negative token strides (which the C entry takes and torch cannot make) give what ascending rows give."""
    dt, dev = DT[dtype], "cuda"
    q, k, v, do = (t.to(dev).contiguous() for t in make(2, 2, 1, tq, tk, d, dt, 7))
    out, lse = layer_ops.attention_forward(q, k, v, True, None, None, None, True)
    want = (out, *layer_ops.attention_backward(q, k, v, out, lse, do, True, None, None, None))
    a = layer_ops.AttentionArgs()
    a.dtype, a.causal, a.bottom_right = {"f32": 0, "f16": 1, "bf16": 2}[dtype], 1, 1
    a.batch, a.heads, a.kv_heads, a.queries, a.keys, a.dim, a.scale = 2, 2, 1, tq, tk, d, d ** -0.5
    held = []

    def place(name, t):  # tokens from the last to the first
        t = t.flip(2).contiguous()
        held.append(t)
        setattr(a, name, t.data_ptr() + (t.shape[2] - 1) * d * t.element_size())
        getattr(a, name + "_stride")[:] = [t.stride(0), t.stride(1), -d]
        return t

    for name, t in (("q", q), ("k", k), ("v", v), ("grad_out", do)):
        place(name, t)
    outs = [place(name, torch.zeros_like(t)) for name, t in (("out", q), ("grad_q", q), ("grad_k", k), ("grad_v", k))]
    log = torch.zeros(2, 2, tq, device=dev)
    a.lse = log.data_ptr()
    lib, stream = N.lib(), torch.cuda.current_stream().cuda_stream
    for step in ("forward", "backward"):
        size = getattr(lib, f"lwl_attention_{step}_workspace_size")(ctypes.byref(a))
        ws = torch.empty(max(size, 1), dtype=torch.uint8, device=dev)
        assert getattr(lib, f"lwl_attention_{step}")(ctypes.byref(a), ws.data_ptr(), size, stream) == 0
    torch.cuda.synchronize()
    for got, ref in zip(outs, want):
        assert torch.allclose(got.flip(2).float(), ref.float(), rtol=0, atol=2 * R.U[dt] * float(ref.abs().max()))


@pytest.mark.parametrize("causal", [False, True])
def test_packed_batch_padded_at_its_ends(causal):
    """Each sequence's tokens see what they see alone, and what pads them takes no part, in both directions."""
    lengths, heads, kv_heads, d = [70, 41, 1, 0, 64], 4, 2, 32
    x = torch.randn(5, 70, (heads + 2 * kv_heads) * d, device="cuda")
    lens = torch.tensor(lengths, device="cuda")
    dy = torch.randn(5, 70, heads * d, device="cuda") * (torch.arange(70, device="cuda")[None] < lens[:, None]).unsqueeze(-1)
    x.requires_grad_()
    y = attention_packed(x, heads, kv_heads, causal=causal, key_lengths=lens)
    (gx,) = torch.autograd.grad(y, x, dy)
    for b, n in enumerate(lengths):
        alone = x[b:b + 1, :n].detach().requires_grad_()
        want = attention_packed(alone, heads, kv_heads, causal=causal)
        (g,) = torch.autograd.grad(want, alone, dy[b:b + 1, :n])
        # the same float32 sums over a sequence's keys in another split at most: some 70 roundings of terms of size 1
        assert torch.allclose(y[b:b + 1, :n], want, rtol=0, atol=1e-5)
        assert torch.allclose(gx[b:b + 1, :n], g, rtol=0, atol=1e-4)
        assert (gx[b, n:] == 0).all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** 100])
def test_the_extreme_scales(dtype, scale):
    """Of scores that are all but equal and of scores that are zero: uniform probabilities, all gradients finite."""
    q, k, v, do = make(1, 2, 1, 40, 70, 64, DT[dtype], 6)
    if scale > 1:
        q = torch.zeros_like(q)
    out, lse = layer_ops.attention_forward(q.cuda(), k.cuda(), v.cuda(), False, scale, None, None, True)
    gq, gk, gv = layer_ops.attention_backward(q.cuda(), k.cuda(), v.cuda(), out, lse, do.cuda(), False, scale, None, None)
    want = v.double().mean(2, keepdim=True).expand_as(out)
    assert (out.double().cpu() - want).abs().max() <= 2 * R.U[DT[dtype]] * 4
    if scale < 1 or dtype != "f16":  # else dQ, 2^100 times sums of size 1, is past the type
        assert torch.isfinite(gq).all()
    assert torch.isfinite(gk).all() and torch.isfinite(gv).all()
