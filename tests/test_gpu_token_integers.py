"""Integers of 64 bits as tokens and parents: what they say holds, also where it does not fit the type that the
kernels read."""
from __future__ import annotations

import pytest
import torch

from conftest import gpu_available
from latent_weight_lab_amd import attention_tree, token_log_probs

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]


def unsigned(values):
    return torch.tensor([v - (1 << 64) if v >= 1 << 63 else v for v in values]).view(torch.uint64).cuda()


def test_unsigned_tokens():
    """From 2^63 on they are past the vocabulary, not none."""
    z = torch.randn(5, 40, device="cuda", requires_grad=True)
    tokens = [3, 39, 40, 1 << 63, (1 << 64) - 1]
    out = token_log_probs(z, unsigned(tokens))
    want = torch.log_softmax(z.detach(), 1)
    assert (out[:2] - torch.stack([want[0, 3], want[1, 39]])).abs().max() < 1e-5
    assert out[2:].isnan().all()
    (dz,) = torch.autograd.grad(out, z, torch.ones(5, device="cuda"))
    (same,) = torch.autograd.grad(token_log_probs(z, torch.tensor([3, 39, 40, 40, 40], device="cuda")), z,
                                  torch.ones(5, device="cuda"))
    assert torch.equal(dz, same) and (dz[2:] == 0).all()


@pytest.mark.parametrize("nodes", [9, 40])
def test_unsigned_parents(nodes):
    """Numbers that are no node's are a root's."""
    q, k, v = (torch.randn(2, 2, n, 32, device="cuda") for n in (nodes, 90, 90))
    parents = torch.arange(nodes) - 1
    parents[[0, 2, 4, 6, 8]] = -1
    no_node = [(1 << 64) - 1, (1 << 32) + 1, 1 << 63, (1 << 63) + 2, (1 << 64) - (1 << 32) + 3]
    given = parents.tolist()
    for at, n in zip((0, 2, 4, 6, 8), no_node):
        given[at] = n
    want = attention_tree(q, k, v, parents.cuda())
    assert torch.equal(attention_tree(q, k, v, unsigned(given)), want)
    assert torch.equal(attention_tree(q, k, v, torch.tensor([p & 0xffffffff for p in parents.tolist()]).to(torch.uint32).cuda()), want)
