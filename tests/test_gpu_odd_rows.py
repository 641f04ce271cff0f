"""Attention of head sizes that are no multiples of eight, at the ends of rows, of tiles of 64 and of tensors: values read
past a row's end must not reach a result."""
from __future__ import annotations

import pytest
import torch

import test_gpu_attention_tree as tree
import test_gpu_attention_window as window
from conftest import gpu_available
from latent_weight_lab_amd import attention, attention_tree
from test_gpu_attention import DT, make

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]

SIZES = [1, 3, 7, 9, 31, 33, 79, 97, 121]


def gapped(t):
    """The same values at an odd address, NaN between rows and after the last one's end."""
    b, h, n, d = t.shape
    buf = torch.full((b * h * n * (d + 3) + 9,), float("nan"), dtype=t.dtype, device="cuda")
    view = buf[1:].as_strided((b, h, n, d), (h * n * (d + 3), n * (d + 3), d + 3, 1), 1)
    view.copy_(t)
    return view


def ending(t):
    """Dense, tokens before heads, the last row at the end of its tensor; rows of other heads are NaN."""
    b, h, n, d = t.shape
    buf = torch.full((b, n, 2 * h, d), float("nan"), dtype=t.dtype, device="cuda")
    view = buf[:, :, h:].transpose(1, 2)
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("dim", SIZES)
@pytest.mark.parametrize("tq,tk", [(1, 1), (40, 2), (63, 63), (64, 64), (65, 65), (20, 130), (191, 129)])
def test_rows_and_their_gradients(dtype, dim, tq, tk):
    dt = DT[dtype]
    q, k, v, do = make(2, 2, 1, tq, tk, dim, dt, dim + tk)
    window.run(q, k, v, do, dt, 50, 3)

    def step(view):
        x = [view(t.cuda()).requires_grad_() for t in (q, k, v)]
        o = attention(*x, causal=True, window=50, sinks=3)
        return [o, *torch.autograd.grad(o, x, view(do.cuda()))]

    want = step(lambda t: t.contiguous())
    for view in (gapped, ending):
        assert all(torch.equal(a, b) for a, b in zip(step(view), want))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("dim", SIZES)
@pytest.mark.parametrize("nodes,tk", [(20, 20), (40, 64), (60, 65), (70, 191), (50, 1600)])
def test_trees(dtype, dim, nodes, tk):
    dt = DT[dtype]
    q, k, v, _ = make(2, 2, 1, nodes, tk, dim, dt, dim + tk)
    parents = tree.some_tree(nodes, 2, nodes)
    tree.run(q, k, v, dt, parents, [tk, max(1, tk - 37)])
    lens = torch.tensor([tk, max(1, tk - 37)], dtype=torch.int32, device="cuda")
    up = torch.tensor(parents, device="cuda")
    q, k, v = (t.cuda() for t in (q, k, v))
    want = attention_tree(q, k.contiguous(), v.contiguous(), up, lens)
    for view in (gapped, ending):
        assert torch.equal(attention_tree(view(q), view(k), view(v), up, lens), want)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("dim,pitch", [(5, 0), (5, 3), (65, 0), (65, 7)])
def test_rows_that_overlap(dtype, dim, pitch):
    """Tokens closer than eight values, all the same one with a stride of 0."""
    dt = DT[dtype]
    buf = torch.randn(70 * 7 + 70, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(dt)
    k, v = (buf[i:].as_strided((1, 1, 70, dim), (0, 0, pitch, 1), i) for i in (0, 1))
    q = torch.randn(1, 2, 70, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).to(dt)
    want = attention(q, k.contiguous(), v.contiguous(), causal=True, window=20)
    assert torch.equal(attention(q, k, v, causal=True, window=20), want)
    up = torch.arange(70, device="cuda") - 1
    assert torch.equal(attention_tree(q, k, v, up), attention_tree(q, k.contiguous(), v.contiguous(), up))
