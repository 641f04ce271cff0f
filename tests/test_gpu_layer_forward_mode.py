"""The layer operators have no forward-mode derivatives and say so: a dropped tangent would be a derivative of zero."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from conftest import gpu_available
from latent_weight_lab_amd import attention, attention_packed, gelu_checkpoint8, gelu_linear_checkpoint8, layer_norm

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]


def dual(*shape):
    t = torch.randn(*shape, device="cuda")
    return forward_ad.make_dual(t, torch.ones_like(t))


CALLS = {
    "norm": lambda: layer_norm(dual(4, 64), torch.ones(64, device="cuda")),
    "norm's weight": lambda: layer_norm(torch.randn(4, 64, device="cuda"), dual(64)),
    "norm's residual": lambda: layer_norm(torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda"),
                                          residual=dual(4, 64)),
    "gelu": lambda: gelu_checkpoint8(dual(4, 64)),
    "gelu's bias": lambda: gelu_checkpoint8(torch.randn(4, 64, device="cuda"), dual(64)),
    "gelu and linear": lambda: gelu_linear_checkpoint8(dual(4, 64), torch.nn.Linear(64, 3, device="cuda")),
    "attention": lambda: attention(*(dual(1, 2, 5, 32) for _ in range(3))),
    "attention's values": lambda: attention(*(torch.randn(1, 2, 5, 32, device="cuda") for _ in range(2)), dual(1, 2, 5, 32)),
    "packed attention": lambda: attention_packed(dual(1, 5, 96), 1),
}


@pytest.mark.parametrize("call", list(CALLS))
@pytest.mark.parametrize("recording", [True, False])
def test_a_tangent_is_refused(call, recording):
    with forward_ad.dual_level(), torch.set_grad_enabled(recording):
        with pytest.raises(NotImplementedError):
            CALLS[call]()


@pytest.mark.parametrize("op", [lambda x: layer_norm(x, torch.ones(96, device="cuda")), gelu_checkpoint8,
                                lambda x: attention(x[None], x[None], x[None]), lambda x: attention_packed(x, 1)])
def test_a_gradients_tangent_is_refused(op):
    """Forward mode over a backward pass."""
    x = torch.randn(1, 5, 96, device="cuda", requires_grad=True)
    y = op(x)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        torch.autograd.grad(y, x, dual(*y.shape))
