"""Attention within a sliding window whose first tokens stay visible (``attention(window=, sinks=)``,
``lwl_attention_window_*``) against float64, both directions; bounds as in ``test_gpu_attention``."""
from __future__ import annotations

import pytest
import torch

import layer_oracle as R
import token_oracle as T
from conftest import gpu_available
from latent_weight_lab_amd import attention, attention_packed, layer_ops
from test_gpu_attention import DT, compare, make

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]


def run(q, k, v, do, dt, window, sinks, lengths=None, offset=None, scale=None, step=True):
    b, h, tq, d = q.shape
    tk = k.shape[2]
    ok = T.window_allowed(tq, tk, lengths, b, offset, window, sinks)
    res = R.attention(q, k, v, scale or d ** -0.5, ok, do if step else None)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    gq, gk, gv = (t.cuda() for t in (q, k, v))
    out, lse = layer_ops.attention_forward(gq, gk, gv, True, scale, lens, offset, True, window, sinks)
    compare(out, res, "o", dt, 2, res["gamma"])
    some = ok.any(2).unsqueeze(1).expand(-1, h, -1)
    assert (lse.cpu()[~some] == float("-inf")).all()
    if some.any():
        off = (lse.double().cpu() - res["lse"]).abs()[some]
        assert (off <= res["gamma"].squeeze(-1)[some] + 2.0 ** -20 * (1 + res["lse"].abs()[some])).all()
    if step:
        gq, gk, gv = (t.requires_grad_() for t in (gq, gk, gv))
        o = attention(gq, gk, gv, causal=True, scale=scale, key_lengths=lens, causal_offset=offset, window=window, sinks=sinks)
        assert torch.equal(o, out)
        for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(o, (gq, gk, gv), do.cuda())):
            compare(g, res, name, dt, 4, res["gamma_all"])


# batch, heads, key heads, queries, keys, head size
SHAPES = [(1, 1, 1, 1, 1, 1), (2, 3, 3, 1, 70, 64), (1, 2, 1, 40, 40, 7), (2, 2, 1, 64, 64, 32), (1, 2, 2, 129, 129, 33),
          (1, 4, 2, 300, 300, 128), (2, 2, 2, 200, 333, 80), (1, 6, 2, 257, 400, 100), (1, 2, 2, 500, 500, 64),
          (1, 8, 1, 2, 1300, 128), (1, 20, 1, 1, 900, 48), (1, 1, 1, 17, 2100, 64), (2, 1, 1, 300, 31, 24)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (17, 4), (64, 0), (100, 65), (128, 130), (5000, 3)])
def test_step_matches_float64(shape, dtype, window, sinks):
    q, k, v, do = make(*shape, DT[dtype], sum(shape) + window)
    run(q, k, v, do, DT[dtype], window, sinks)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("tq,tk,lengths", [(40, 150, [0, 1, 150, 63, 64, 65]), (200, 200, [200, 0, 5, 128, 129, 199]),
                                           (1, 400, [1, 0, 400, 31, 32, 33]), (4, 1200, [3, 1200, 0, 257, 1, 800])])
@pytest.mark.parametrize("offset", [None, 0, -3, 100, 390])
@pytest.mark.parametrize("window,sinks", [(50, 0), (50, 5), (3, 70)])
def test_lengths_and_offsets(dtype, tq, tk, lengths, offset, window, sinks):
    """Empty and short sequences, queries past every window, with anything at all past the sequences' ends and in queries
    that see nothing."""
    q, k, v, do = make(6, 4, 2, tq, tk, 64, DT[dtype], tq + tk)
    k, v, q, do = k.clone(), v.clone(), q.clone(), do.clone()
    for i, n in enumerate(lengths):
        k[i, :, n:] = float("nan")
        v[i, :, n:] = float("inf")
    none = ~T.window_allowed(tq, tk, lengths, 6, offset, window, sinks).any(2)
    q.permute(0, 2, 1, 3)[none] = float("nan")
    do.permute(0, 2, 1, 3)[none] = float("inf")
    run(q, k, v, do, DT[dtype], window, sinks, lengths=lengths, offset=offset)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 2, 2, 2500, 2500, 64), (1, 8, 2, 1030, 1030, 48), (2, 1, 1, 900, 1700, 128)])
def test_sinks_of_long_sequences(dtype, shape):
    """The key blocks of sinks take far more queries than the others, and are summed from ranges."""
    q, k, v, do = make(*shape, DT[dtype], 3)
    run(q, k, v, do, DT[dtype], 70, 2)
    run(q, k, v, do, DT[dtype], 70, 150)


@pytest.mark.parametrize("dtype", list(DT))
def test_large_batches(dtype):
    """More sequences than a wave has lanes."""
    for tq in (1, 40):
        q, k, v, do = make(70, 2, 1, tq, 300, 32, DT[dtype], tq)
        run(q, k, v, do, DT[dtype], 37, 3, lengths=[(i * 41) % 301 for i in range(70)])


@pytest.mark.parametrize("dtype", list(DT))
def test_a_wide_window_is_none(dtype):
    """A window that hides nothing gives what causal order alone gives, to its rounding."""
    q, k, v, do = (t.cuda() for t in make(2, 4, 2, 150, 200, 64, DT[dtype], 7))
    want = attention(q, k, v, causal=True)
    for window, sinks in ((200, 0), (1 << 40, 0), ((1 << 63) - 1, (1 << 62)), (1, 200)):
        got = attention(q, k, v, causal=True, window=window, sinks=sinks)
        # the same products and sums; tiles may be cut otherwise
        assert (got - want).abs().max() <= 4 * R.U[DT[dtype]] * want.abs().max()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("heads,kv_heads,dim,t", [(4, 4, 64, 100), (6, 2, 40, 277), (3, 1, 9, 33)])
def test_packed_is_the_same(dtype, heads, kv_heads, dim, t):
    dt = DT[dtype]
    g = torch.Generator().manual_seed(t)
    x = torch.randn(2, t, (heads + 2 * kv_heads) * dim, generator=g).to(dt).cuda().requires_grad_()
    dy = torch.randn(2, t, heads * dim, generator=g).to(dt).cuda()
    lens = torch.tensor([t, t // 2], device="cuda")
    for lengths in (None, lens):
        y = attention_packed(x, heads, kv_heads, key_lengths=lengths, window=20, sinks=3)
        (gx,) = torch.autograd.grad(y, x, dy)
        q, k, v = (s.unflatten(-1, (-1, dim)).transpose(1, 2)
                   for s in x.split([heads * dim, kv_heads * dim, kv_heads * dim], -1))
        o = attention(q, k, v, causal=True, key_lengths=lengths, causal_offset=0, window=20, sinks=3)
        o = o.transpose(1, 2).reshape(2, t, -1)
        assert torch.equal(y, o)
        assert torch.equal(gx, torch.autograd.grad(o, x, dy)[0])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_layouts(dtype):
    """Strides of every kind give what contiguous tensors give, bit for bit."""
    dt = DT[dtype]
    q, k, v, do = (t.cuda() for t in make(2, 4, 2, 170, 290, 72, dt, 5))
    how = {"causal": True, "window": 75, "sinks": 6}

    def step(leaves, up):
        leaves = [t.detach().requires_grad_() for t in leaves]
        o = attention(*leaves, **how)
        return [o, *torch.autograd.grad(o, leaves, up)]

    def odd(t):  # odd offset and odd strides
        b, h, n, d = t.shape
        buf = torch.full((b, n, h, d + 5), float("nan"), dtype=dt, device="cuda")
        view = buf[..., 3:3 + d].transpose(1, 2)
        view.copy_(t)
        return view

    want = step([t.contiguous() for t in (q, k, v)], do)
    got = step([odd(t) for t in (q, k, v)], odd(do))
    assert torch.equal(want[0], got[0])
    for a, b in zip(want[1:], got[1:]):
        assert torch.equal(a, b) or (a - b).abs().max() <= 4 * R.U[dt] * a.abs().max()
    # heads that share keys by stride 0
    k1, v1 = k[:, :1], v[:, :1]
    assert torch.equal(attention(q, k1.expand(-1, 4, -1, -1), v1.expand(-1, 4, -1, -1), **how), attention(q, k1, v1, **how))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_tokens_over_a_cache_equal_the_prompt(dtype):
    """One to sixty tokens at a time over a preallocated cache give the rows of the whole prompt's pass."""
    dt = DT[dtype]
    q, k, v, _ = (t.cuda() for t in make(2, 6, 3, 500, 500, 64, dt, 9))
    whole = attention(q, k, v, causal=True, window=90, sinks=4)
    cache_k, cache_v = (torch.full((2, 1024, 3, 64), float("nan"), device="cuda", dtype=dt) for _ in range(2))
    done = 0
    for n in [300, 1, 5, 1, 2, 60, 131]:
        cache_k[:, done:done + n] = k[:, :, done:done + n].transpose(1, 2)
        cache_v[:, done:done + n] = v[:, :, done:done + n].transpose(1, 2)
        lens = torch.full((2,), done + n, device="cuda")
        o = attention(q[:, :, done:done + n], cache_k.transpose(1, 2), cache_v.transpose(1, 2), causal=True,
                      key_lengths=lens, window=90, sinks=4)
        # float32: other orders of the same sums.  bfloat16: the probabilities are rounded relative to another
        # maximum, half a step of each of them and of the result, in both passes
        bound = 1e-5 if dtype == "f32" else 4 * R.U[dt] * v.abs().max().item()
        assert (o - whole[:, :, done:done + n]).abs().max() < bound
        done += n


def test_hidden_keys_far_away_are_not_read():
    """NaN in keys and values that no query of a block sees reaches nothing."""
    q, k, v, do = (t.cuda() for t in make(1, 2, 2, 40, 3000, 64, torch.bfloat16, 4))
    want = attention(q, k, v, causal=True, window=100, sinks=5)
    k2, v2 = k.clone(), v.clone()
    k2[:, :, 5:2860] = float("nan")  # queries 2960 .. 2999 see 2861 and up
    v2[:, :, 5:2860] = float("nan")
    assert torch.equal(attention(q, k2, v2, causal=True, window=100, sinks=5), want)
    assert torch.equal(attention(q[:, :, -1:], k2, v2, causal=True, window=100, sinks=5),
                       attention(q[:, :, -1:], k, v, causal=True, window=100, sinks=5))
    leaves = [t.detach().requires_grad_() for t in (q, k2, v2)]
    grads = torch.autograd.grad(attention(*leaves, causal=True, window=100, sinks=5), leaves, do)
    assert all(torch.isfinite(g).all() for g in grads)
    assert (grads[1][:, :, 5:2860] == 0).all() and (grads[2][:, :, 5:2860] == 0).all()


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
        how = {"causal": True, "window": 70, "sinks": 3}
        assert torch.equal(attention(q[:, :, :n], bk, bv, **how), attention(q[:, :, :n], k, v, **how))


def test_extreme_scores():
    for dt in DT.values():
        q = torch.zeros(1, 1, 300, 64, dtype=dt)
        k = torch.zeros(1, 1, 300, 64, dtype=dt)
        v = torch.randn(1, 1, 300, 64, generator=torch.Generator().manual_seed(1)).to(dt)
        q[..., 0] = 100.0
        k[0, 0, :, 0] = torch.linspace(-200.0, 200.0, 300).to(dt)
        for kk in (k, k.flip(2)):
            run(q, kk, v, v.clone(), dt, 40, 3)


def test_repeats_streams_and_graph():
    q, k, v, do = (t.cuda() for t in make(2, 6, 2, 700, 700, 64, torch.bfloat16, 8))
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    how = {"causal": True, "window": 100, "sinks": 4}

    def step():
        o = attention(*leaves, **how)
        return [o, *torch.autograd.grad(o, leaves, do)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    ck, cv = (torch.randn(2, 2000, 2, 64, device="cuda").bfloat16().transpose(1, 2) for _ in range(2))
    lens = torch.tensor([5, 7], dtype=torch.int32, device="cuda")
    q1 = q[:, :, :1].contiguous()
    graph = torch.cuda.CUDAGraph()
    attention(q1, ck, cv, key_lengths=lens, **how)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        o = attention(q1, ck, cv, key_lengths=lens, **how)
    for n in (5, 2000, 900, 1):
        lens.fill_(n)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, attention(q1, ck, cv, key_lengths=lens, **how))


def test_refusals():
    q = torch.randn(2, 4, 8, 32, device="cuda")
    k = torch.randn(2, 2, 9, 32, device="cuda")
    for bad in (lambda: attention(q, k, k, window=4), lambda: attention(q, k, k, causal=True, window=0),
                lambda: attention(q, k, k, causal=True, window=-5), lambda: attention(q, k, k, causal=True, sinks=2),
                lambda: attention(q, k, k, causal=True, window=3, sinks=-1), lambda: attention(q, k, k, causal=True, window=2.5)):
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            bad()


@pytest.mark.parametrize("tq,tk,b", [(0, 5, 2), (3, 0, 2), (0, 0, 1), (4, 6, 0)])
def test_empty_tensors(tq, tk, b):
    q = torch.randn(b, 4, tq, 32, device="cuda", requires_grad=True)
    k = torch.randn(b, 2, tk, 32, device="cuda", requires_grad=True)
    v = torch.randn(b, 2, tk, 32, device="cuda", requires_grad=True)
    o = attention(q, k, v, causal=True, window=3, sinks=1)
    assert o.shape == q.shape and (o == 0).all()
    for g, t in zip(torch.autograd.grad(o.sum(), (q, k, v)), (q, k, v)):
        assert g.shape == t.shape and (g == 0).all()
