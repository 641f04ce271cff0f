"""Rows of ``token_log_probs``: none at all in any layout, and more than a grid's axis has workgroups."""
from __future__ import annotations

import pytest
import torch

from conftest import gpu_available
from layer_oracle import U
from latent_weight_lab_amd import token_log_probs

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]


@pytest.mark.parametrize("empty", [0, 1, 2])
def test_no_rows_of_axes_that_lie_apart(empty):
    z = torch.randn(4, 6, 8, 20, device="cuda")[::2, :5, :7].narrow(empty, 0, 0).requires_grad_()
    rows = z.shape[:-1]
    tokens = torch.zeros(rows, dtype=torch.long, device="cuda")
    out = token_log_probs(z, tokens, entropy=True, top=2)
    assert [o.shape for o in out] == [rows, rows, (*rows, 2), (*rows, 2)]
    (dz,) = torch.autograd.grad([out[0].sum(), out[1].sum()], z)
    assert dz.shape == z.shape


@pytest.mark.parametrize("rows", [(1 << 22) + 1, (1 << 24) + 3])
def test_more_rows_than_workgroups(rows):
    """Both directions of rows of three tokens.  The results are sums of three terms of logits below 4: off by less than 2^-20, and
    the gradients, below 1, rounded to the type."""
    g = torch.Generator(device="cuda").manual_seed(7)
    z = torch.rand(rows, 3, device="cuda", generator=g).mul(4).bfloat16().requires_grad_()
    tokens = torch.randint(3, (rows,), device="cuda", generator=g)
    out = token_log_probs(z, tokens)
    want = torch.log_softmax(z.detach().double(), 1)
    assert (out - want.gather(1, tokens[:, None])[:, 0]).abs().max() < 2.0 ** -20
    (dz,) = torch.autograd.grad(out, z, torch.ones_like(out))
    grad = torch.nn.functional.one_hot(tokens, 3) - want.exp()
    assert (dz - grad).abs().max() < U[torch.bfloat16] + 2.0 ** -19
