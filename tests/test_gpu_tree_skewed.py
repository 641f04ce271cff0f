"""Batches in which one sequence is much longer than the others: it then has most of the ranges, many more than the average
that the join is laid out for."""
from __future__ import annotations

import pytest
import torch

from conftest import gpu_available
from latent_weight_lab_amd import attention_tree
from test_gpu_attention import DT, make
from test_gpu_attention_tree import run, some_tree

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]


# batch, heads, key heads, nodes, keys, head size: a join of 16 threads a chunk, of 4 and of 1; single tokens' kernel
@pytest.mark.parametrize("shape", [(20, 1, 1, 20, 12_000, 64), (3, 2, 1, 18, 20_000, 32), (40, 8, 2, 20, 4000, 40),
                                   (20, 4, 1, 3, 9000, 33), (64, 1, 1, 1, 6000, 128)])
@pytest.mark.parametrize("dtype", list(DT))
def test_one_long_sequence(shape, dtype):
    b, _, _, n, tk, _ = shape
    q, k, v, _ = make(*shape, DT[dtype], sum(shape))
    lengths = [(17 * i) % (n + 60) for i in range(b)]
    lengths[b // 2] = tk
    run(q, k, v, DT[dtype], some_tree(n, b, n), lengths)


def test_what_others_have_does_not_count():
    """A sequence's results are the same, but for the order of sums, whatever ranges the batch leaves it."""
    q, k, v, _ = (t.cuda() for t in make(64, 4, 1, 32, 8192, 64, torch.float32, 3))
    parents = torch.tensor(some_tree(32, 64, 2), device="cuda")
    full = torch.full((64,), 8192, device="cuda")
    one = torch.full((64,), 40, device="cuda")
    one[5] = 8192
    a, b = (attention_tree(q, k, v, parents, n) for n in (full, one))
    # sums of values below 6, probabilities that sum to 1, each range's rounded a few times
    assert (a[5] - b[5]).abs().max() < 6 * 32 * 2.0 ** -24
