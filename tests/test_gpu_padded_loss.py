"""The mean of a loss over targets of which some are padding, as torch's cross entropy takes it."""
import pytest
import torch
import torch.nn.functional as F

from latent_weight_lab_amd import token_log_probs
from test_gpu_gpt2_stack import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("padding", [-1, -100])
def test_mean_over_targets(padding):
    """As the documentation gives it.  Float32: 300 terms of about log 1000 and a division, each off by 2^-24 of its size."""
    z = torch.randn(3, 100, 1000, device="cuda", requires_grad=True)
    targets = torch.randint(1000, (3, 100), device="cuda")
    targets[0, 40:] = targets[2, :95] = padding
    loss = -token_log_probs(z, targets).sum() / (targets >= 0).sum()
    (dz,) = torch.autograd.grad(loss, z)
    z64 = z.detach().double().requires_grad_()
    want = F.cross_entropy(z64.flatten(0, 1), targets.flatten(), ignore_index=padding)
    (d64,) = torch.autograd.grad(want, z64)
    assert abs(loss.item() - want.item()) < 300 * 2.0 ** -24 * want.item()
    assert (dz - d64).abs().max() < 2.0 ** -20 * d64.abs().max()


class Still:
    """An optimizer that leaves everything as it is."""

    def __init__(self, model):
        self.model = model

    def zero_grad(self, set_to_none):
        self.model.zero_grad(set_to_none=set_to_none)

    def step(self):
        pass


def test_a_stacks_step_leaves_padding_out():
    """The loss and every gradient are those of the targets that are there: of a batch, and of one whose other sequence is
    nothing but padding."""
    model = make()
    ids = torch.randint(131, (2, 41), device="cuda")
    x, y = ids[:, :-1].contiguous(), ids[:, 1:].contiguous()
    alone = model.step(x[:1], y[:1], Still(model))
    grads = [p.grad.clone() for p in model.parameters()]
    for padding in (-100, -1):
        padded = y.clone()
        padded[1] = padding
        loss = model.step(x, padded, Still(model))
        # the same sums, the second sequence's zeros among them, in another order: some 2^-24 of each of 40 terms
        assert abs(loss.item() - alone.item()) < 1e-5 * alone.item()
        for p, g in zip(model.parameters(), grads):
            # a code of an 8-bit checkpoint may fall to its neighbour, 1 of 127 steps of its scale: below that even if all did
            assert (p.grad - g).norm() <= 0.02 * g.norm()
