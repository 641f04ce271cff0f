"""Attention of a tree of drafted tokens over a cache (``attention_tree``, ``lwl_attention_tree_forward``) against float64;
bounds as in ``test_gpu_attention``."""
from __future__ import annotations

import ctypes

import pytest
import torch

import layer_oracle as R
import token_oracle as T
from conftest import gpu_available
from latent_weight_lab_amd import _native as N
from latent_weight_lab_amd import attention, attention_tree, layer_ops
from test_gpu_attention import DT, compare, make

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]


def some_tree(nodes, batch, seed, kind="any"):
    g = torch.Generator().manual_seed(seed)
    if kind == "chain":
        return [[i - 1 for i in range(nodes)] for _ in range(batch)]
    if kind == "roots":
        return [[-1] * nodes for _ in range(batch)]
    return [[int(torch.randint(-1, i, (1,), generator=g)) if i else -1 for i in range(nodes)] for _ in range(batch)]


def run(q, k, v, dt, parents, lengths=None, scale=None):
    b, h, n, d = q.shape
    ok = T.tree_allowed(parents, k.shape[2], lengths, b)
    res = R.attention(q, k, v, scale or d ** -0.5, ok)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = attention_tree(q.cuda(), k.cuda(), v.cuda(), torch.tensor(parents, device="cuda"), lens, scale)
    compare(out, res, "o", dt, 2, res["gamma"])
    assert out.transpose(1, 2).is_contiguous()
    return out


# batch, heads, key heads, nodes, keys, head size: one node, up to 16 rows on a key head, more, several blocks of 128
# rows, nodes that cross tiles, ranges of a long cache
SHAPES = [(1, 1, 1, 1, 1, 1), (2, 3, 3, 1, 64, 64), (1, 2, 2, 16, 40, 32), (2, 8, 2, 4, 300, 64), (1, 4, 1, 5, 70, 33),
          (3, 4, 2, 17, 81, 80), (1, 8, 2, 32, 700, 128), (2, 2, 2, 33, 64, 7), (1, 2, 1, 64, 64, 64), (2, 2, 2, 65, 200, 96),
          (1, 3, 1, 100, 1000, 64), (1, 6, 2, 128, 333, 100), (1, 4, 1, 128, 2100, 128), (1, 20, 1, 7, 900, 48),
          (1, 2, 2, 11, 3000, 64)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("kind", ["any", "chain", "roots"])
def test_matches_float64(shape, dtype, kind):
    q, k, v, _ = make(*shape, DT[dtype], sum(shape))
    run(q, k, v, DT[dtype], some_tree(shape[3], shape[0], sum(shape), kind))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("nodes,tk,lengths", [(5, 150, [0, 1, 150, 5, 64, 65]), (40, 200, [200, 0, 5, 40, 129, 39]),
                                              (100, 260, [100, 260, 0, 63, 101, 228]), (4, 1200, [3, 1200, 0, 257, 1, 800])])
def test_lengths(dtype, nodes, tk, lengths):
    """Sequences shorter than the tree, and with anything at all past their ends."""
    q, k, v, _ = make(6, 4, 2, nodes, tk, 64, DT[dtype], nodes + tk)
    k, v = k.clone(), v.clone()
    for i, n in enumerate(lengths):
        k[i, :, n:] = float("nan")
        v[i, :, n:] = float("inf")
    parents = some_tree(nodes, 6, nodes)
    q = q.clone()
    q.permute(0, 2, 1, 3)[~T.tree_allowed(parents, tk, lengths, 6).any(2)] = float("nan")
    run(q, k, v, DT[dtype], parents, lengths)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("heads,nodes,tk", [(2, 32, 31), (2, 32, 32), (2, 32, 33), (1, 64, 95), (1, 64, 96), (1, 17, 97),
                                            (4, 9, 1024 + 31), (1, 33, 2048 + 33)])
def test_halves_of_a_tile(dtype, heads, nodes, tk):
    """Up to 64 rows: sequences that end in either half of 64 keys; scores of one half far above the other's, either way."""
    q, k, v, _ = make(4, heads, 1, nodes, tk, 40, DT[dtype], heads + nodes + tk)
    lengths = [tk, max(0, tk - 32), tk, tk - 1]
    k = k.clone()
    q = q.clone()
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    k[0, :, torch.arange(tk) % 64 < 32, 0] = 4.0
    k[2, :, torch.arange(tk) % 64 >= 32, 0] = 4.0
    parents = some_tree(nodes, 4, nodes)
    q.permute(0, 2, 1, 3)[~T.tree_allowed(parents, tk, lengths, 4).any(2)] = float("nan")
    run(q, k, v, DT[dtype], parents, lengths, 1.0)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("nodes", [3, 40])
def test_a_chain_is_causal(dtype, nodes):
    q, k, v, _ = (t.cuda() for t in make(2, 4, 2, nodes, 500, 64, DT[dtype], 1))
    chain = torch.arange(nodes, device="cuda") - 1
    for lens in (None, torch.tensor([nodes, 333], device="cuda")):
        got, want = attention_tree(q, k, v, chain, lens), attention(q, k, v, causal=True, key_lengths=lens)
        # the same scores; probabilities relative to other maxima, rounded in both, and the results
        assert (got - want).abs().max() <= 4 * R.U[DT[dtype]] * v.abs().max()


@pytest.mark.parametrize("nodes", [9, 50])
def test_parents_that_are_no_nodes(nodes):
    """Numbers outside of the nodes before make roots; every integer type; one tree for all."""
    q, k, v, _ = (t.cuda() for t in make(2, 2, 1, nodes, 100, 32, torch.bfloat16, 6))
    parents = torch.tensor(some_tree(nodes, 2, 5))
    want = attention_tree(q, k, v, parents.cuda())
    odd = parents.clone()
    roots = odd == -1
    odd[roots] = torch.tensor([1 << 40, -(1 << 40), nodes, 127, 128, 1 << 32, (1 << 32) - 1, -(1 << 31)])[
        torch.arange(int(roots.sum())) % 8]
    odd[:, 4] = 4  # itself
    parents[:, 4] = -1
    want = attention_tree(q, k, v, parents.cuda())
    assert torch.equal(attention_tree(q, k, v, odd.cuda()), want)
    for t in (torch.int32, torch.int16, torch.int8):
        assert torch.equal(attention_tree(q, k, v, parents.to(t).cuda()), want)
    one = attention_tree(q, k, v, parents[1].cuda())
    assert torch.equal(one, attention_tree(q, k, v, parents[1:].expand(2, -1).cuda()))
    assert torch.equal(one[1], want[1])
    # columns of a larger table
    table = torch.full((2, nodes + 3), -1)
    table[:, 2:2 + nodes] = parents
    assert torch.equal(attention_tree(q, k, v, table.cuda()[:, 2:2 + nodes]), want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nodes", [3, 30])
def test_layouts(dtype, nodes):
    dt = DT[dtype]
    q, k, v, _ = (t.cuda() for t in make(2, 4, 2, nodes, 290, 72, dt, 5))
    parents = torch.tensor(some_tree(nodes, 2, 5), device="cuda")
    want = attention_tree(q.contiguous(), k.contiguous(), v.contiguous(), parents)

    def odd(t):  # odd offset and odd strides
        b, h, n, d = t.shape
        buf = torch.full((b, n, h, d + 5), float("nan"), dtype=dt, device="cuda")
        view = buf[..., 3:3 + d].transpose(1, 2)
        view.copy_(t)
        return view

    for make_view in (lambda t: t, odd, lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(attention_tree(*(make_view(t) for t in (q, k, v)), parents), want)
    k1, v1 = k[:, :1], v[:, :1]
    got = attention_tree(q, k1.expand(-1, 4, -1, -1), v1.expand(-1, 4, -1, -1), parents)
    assert (got - attention_tree(q, k1, v1, parents)).abs().max() <= 4 * R.U[dt] * v.abs().max()


def test_offsets_past_32_bits():
    """A cache whose tokens lie more than 2^31 values apart."""
    stride = (1 << 31) // 300 + 64
    buf = torch.zeros(stride * 400, dtype=torch.float16, device="cuda")
    q, k, v, _ = (t.cuda() for t in make(1, 1, 1, 60, 400, 64, torch.float16, 2))
    bk = buf.as_strided((1, 1, 400, 64), (0, 0, stride, 1))
    bv = buf[128:].as_strided((1, 1, 400, 64), (0, 0, stride, 1))
    bk.copy_(k)
    bv.copy_(v)
    parents = torch.tensor(some_tree(60, 1, 2)[0], device="cuda")
    for n in (60, 3):
        assert torch.equal(attention_tree(q[:, :, :n], bk, bv, parents[:n]), attention_tree(q[:, :, :n], k, v, parents[:n]))


@pytest.mark.parametrize("nodes,d,hk", [(4, 64, 2), (40, 32, 1)])
def test_large_batches(nodes, d, hk):
    """More sequences than a wave has lanes, and as many, of all lengths."""
    for b in (64, 65, 130):
        q, k, v, _ = make(b, 2, hk, nodes, 600, d, torch.bfloat16, b)
        lengths = [(i * 97) % 601 for i in range(b)]
        run(q, k, v, torch.bfloat16, some_tree(nodes, b, b), lengths)


@pytest.mark.parametrize("nodes,d", [(2, 64), (30, 128)])
def test_log_sums_of_the_c_entry(nodes, d):
    """lse, which only C callers ask for, from one range and from several."""
    for tk in (100, 3000):
        q, k, v, _ = make(2, 4, 2, nodes, tk, d, torch.float16, 3)
        parents = some_tree(nodes, 2, 1)
        lengths = [tk, nodes - 1]
        ok = T.tree_allowed(parents, tk, lengths, 2)
        res = R.attention(q, k, v, d ** -0.5, ok)
        q, k, v = (t.cuda().contiguous() for t in (q, k, v))
        out, lse = torch.empty_like(q), torch.empty(2, 4, nodes, device="cuda")
        lens, par = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in (lengths, parents))
        a = layer_ops.AttentionArgs()
        a.dtype, a.batch, a.heads, a.kv_heads, a.queries, a.keys, a.dim, a.scale = 1, 2, 4, 2, nodes, tk, d, d ** -0.5
        a.q, a.k, a.v, a.out, a.lse, a.key_lengths = (t.data_ptr() for t in (q, k, v, out, lse, lens))
        for f, t in (("q_stride", q), ("k_stride", k), ("v_stride", v), ("out_stride", out)):
            for i in range(3):
                getattr(a, f)[i] = t.stride(i)
        need = N.lib().lwl_attention_tree_workspace_size(ctypes.byref(a))
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        N.check(N.lib().lwl_attention_tree_forward(ctypes.byref(a), par.data_ptr(), nodes, ws.data_ptr(), need,
                                                   torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        compare(out, res, "o", torch.float16, 2, res["gamma"])
        some = ok.any(2).unsqueeze(1).expand(-1, 4, -1)
        assert (lse.cpu()[~some] == float("-inf")).all()
        off = (lse.double().cpu() - res["lse"]).abs()[some]
        assert (off <= res["gamma"].squeeze(-1)[some] + 2.0 ** -20 * (1 + res["lse"].abs()[some])).all()


def test_streams_and_graphs():
    """Two captured graphs in turn, the lengths and the tree read on the device."""
    ck, cv = (torch.randn(2, 2000, 2, 64, device="cuda").bfloat16().transpose(1, 2) for _ in range(2))
    for nodes in (6, 40):
        q = torch.randn(2, 4, nodes, 64, device="cuda").bfloat16()
        graphs = []
        for _ in range(2):
            lens = torch.tensor([nodes, 50], dtype=torch.int32, device="cuda")
            parents = torch.full((2, nodes), -1, dtype=torch.int32, device="cuda")
            attention_tree(q, ck, cv, parents, lens)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                o = attention_tree(q, ck, cv, parents, lens)
            graphs.append((graph, o, lens, parents))
        for n in (nodes, 2000, 900, nodes + 1):
            for i, (graph, o, lens, parents) in enumerate(graphs):
                lens.fill_(n)
                parents.copy_(torch.tensor(some_tree(nodes, 2, n + i)))
                graph.replay()
                torch.cuda.synchronize()
                want = attention_tree(q, ck, cv, parents, lens)
                assert torch.equal(o, want)
                side = torch.cuda.Stream()
                with torch.cuda.stream(side):
                    again = attention_tree(q, ck, cv, parents, lens)
                side.synchronize()
                assert torch.equal(again, want)


def test_refusals():
    q = torch.randn(2, 4, 8, 32, device="cuda")
    k = torch.randn(2, 2, 9, 32, device="cuda")
    p = torch.zeros(2, 8, dtype=torch.int32, device="cuda")
    attention_tree(q, k, k, p)
    long_q = torch.randn(2, 4, 129, 32, device="cuda")
    for bad in (lambda: attention_tree(q, k, k, p[:, :7]), lambda: attention_tree(q, k, k, p[:1]), lambda: attention_tree(q, k, k, p.float()),
                lambda: attention_tree(q, k, k, p.cpu()), lambda: attention_tree(q, k, k, p[None]),
                lambda: attention_tree(long_q, k, k, torch.zeros(129, dtype=torch.int32, device="cuda")),
                lambda: attention_tree(q, k, k.half(), p), lambda: attention_tree(q, k[:, :, :, :31], k, p),
                lambda: attention_tree(q, k, k, p, scale=0.0), lambda: attention_tree(q[:, :3], k, k, p),
                lambda: attention_tree(q, k, k, p, p[0]), lambda: attention_tree(q.cpu(), k.cpu(), k.cpu(), p.cpu())):
        with pytest.raises((RuntimeError, ValueError)):
            bad()
    leaf = q.clone().requires_grad_()
    with pytest.raises(NotImplementedError):
        attention_tree(leaf, k, k, p)
    with torch.no_grad():
        attention_tree(leaf, k, k, p)


@pytest.mark.parametrize("nodes,tk,b", [(0, 5, 2), (3, 0, 2), (0, 0, 1), (4, 6, 0)])
def test_empty_tensors(nodes, tk, b):
    q, k = torch.randn(b, 4, nodes, 32, device="cuda"), torch.randn(b, 2, tk, 32, device="cuda")
    o = attention_tree(q, k, k, torch.full((b, nodes), -1, device="cuda"))
    assert o.shape == q.shape and (o == 0).all()
