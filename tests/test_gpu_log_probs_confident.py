"""The entropy of rows in which one token has nearly all probability."""
from __future__ import annotations

import pytest
import torch

from conftest import gpu_available
from layer_oracle import EPS32
from latent_weight_lab_amd import token_log_probs
from test_gpu_log_probs import DT

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("vocab,threads,top", [(4096, 256, 0), (4096, 256, 3), (32_768, 512, 0), (32_768, 512, 3)])
def test_entropies_of_confident_rows(dtype, vocab, threads, top):
    """A thread meets a value 4 to 8 below the row's largest in its first chunk of eight, the largest as the last of its second,
    and nothing else counts.

    Let u be float32's roundoff, g the distance and s = exp(-g).  The largest value's own term is exactly 1, s is off by
    (3 g + 4) u of itself (the difference, its product with log2(e), the instruction), less than 28 u, and 1 + s is rounded
    once, by u; what is added later, exp(-40) times a row's length, leaves 1 + s as it is.  So log S is off by u + 28 u s, and by 3 u of
    its value, which is below s.  Where the terms of A = sum e^d d are all below 0, A = -g s is off by 34 u of itself, A / S
    by 36 u and the difference by one more.  The entropy H = log S - A / S is at least (1 + g) s (1 - s) > 4.9 s: together
    u + 31 u s + 37 u H < u + 44 u H."""
    dt, rows = DT[dtype], 256
    g = torch.Generator().manual_seed(vocab + top)
    z = torch.full((rows, vocab), -40.0)
    thread = torch.randint(threads, (rows,), generator=g)
    row = torch.arange(rows)
    z[row, thread * 8 + torch.randint(8, (rows,), generator=g)] = -4 - 3.95 * torch.rand(rows, generator=g)
    z[row, (threads + thread) * 8 + 7] = 0.0
    z = z.to(dt)
    lp = torch.log_softmax(z.double(), 1)
    want = -(lp.exp() * lp).sum(1)
    tokens = z.argmax(1)
    out = token_log_probs(z.cuda(), tokens.cuda(), entropy=True, top=top)
    off = (out[1].double().cpu() - want).abs()
    assert (off <= EPS32 + 44 * EPS32 * want).all(), (off / EPS32).max().item()
