"""Windows, drafted trees and log probabilities in forward mode, which they refuse, and in a training step captured into a
graph."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from conftest import gpu_available
from latent_weight_lab_amd import attention, attention_packed, attention_tree, token_log_probs

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]


def dual(*shape):
    t = torch.randn(*shape, device="cuda")
    return forward_ad.make_dual(t, torch.ones_like(t))


def plain(*shape):
    return torch.randn(*shape, device="cuda")


PARENTS = [-1, 0, 0, 1, 2]
CALLS = {
    "log probabilities": lambda: token_log_probs(dual(4, 64), torch.zeros(4, dtype=torch.long, device="cuda"), entropy=True),
    "window": lambda: attention(*(dual(1, 2, 5, 32) for _ in range(3)), causal=True, window=2),
    "window's values": lambda: attention(plain(1, 2, 5, 32), plain(1, 2, 5, 32), dual(1, 2, 5, 32), causal=True, window=2),
    "packed window": lambda: attention_packed(dual(1, 5, 96), 1, window=2, sinks=1),
    "tree": lambda: attention_tree(*(dual(1, 2, 5, 32) for _ in range(3)), torch.tensor(PARENTS, device="cuda")),
    "tree's keys": lambda: attention_tree(plain(1, 2, 5, 32), dual(1, 2, 5, 32), plain(1, 2, 5, 32),
                                          torch.tensor(PARENTS, device="cuda")),
}


@pytest.mark.parametrize("call", list(CALLS))
@pytest.mark.parametrize("recording", [True, False])
def test_a_tangent_is_refused(call, recording):
    with forward_ad.dual_level(), torch.set_grad_enabled(recording):
        with pytest.raises(NotImplementedError):
            CALLS[call]()


@pytest.mark.parametrize("op", [lambda x: token_log_probs(x, torch.zeros(1, 5, dtype=torch.long, device="cuda")),
                                lambda x: attention_packed(x, 1, window=3)])
def test_a_gradients_tangent_is_refused(op):
    """Forward mode over a backward pass."""
    x = torch.randn(1, 5, 96, device="cuda", requires_grad=True)
    y = op(x)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        torch.autograd.grad(y, x, dual(*y.shape))


@pytest.mark.parametrize("op", ["window", "log probabilities"])
def test_a_captured_step(op):
    """Forward and backward in one graph, replayed with new inputs between eager work of other tensors."""
    g = torch.Generator().manual_seed(5)
    if op == "window":
        x = torch.randn(2, 700, 3 * 128, generator=g).bfloat16().cuda().requires_grad_()
        up = torch.randn(2, 700, 128, generator=g).bfloat16().cuda()

        def step(x):
            y = attention_packed(x, 2, window=60, sinks=3)
            return y.detach(), torch.autograd.grad(y, x, up)[0]
    else:
        x = torch.randn(50, 9001, generator=g).cuda().requires_grad_()
        up = torch.randn(50, generator=g).cuda()
        tokens = torch.randint(9001, (50,), generator=g).cuda()

        def step(x):
            lp, h, top, index = token_log_probs(x, tokens, entropy=True, top=3)
            return lp.detach(), h.detach(), top.detach(), index, torch.autograd.grad([lp, h], x, [up, up])[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x)
    for _ in range(4):
        new = torch.randn(x.shape, generator=g).to(x.dtype).cuda()
        with torch.no_grad():
            x.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        want = step(new.requires_grad_())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
