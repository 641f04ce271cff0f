"""The alternatives of ``token_log_probs`` where a few threads hold many of a row's largest values: they then pass over the row
again, and drop all but the largest whenever the next values may not fit."""
from __future__ import annotations

import pytest
import torch

from conftest import gpu_available
from test_gpu_log_probs import DT, run

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]


def crowded(vocab, threads, dt, kind):
    """Large values in all chunks of eight of the first 63 of `threads` threads, smaller ones in the 64th's, so that with 64
    alternatives each of these passes the bound: 504 values a round, of 1024 that fit."""
    g = torch.Generator().manual_seed(vocab)
    z = torch.rand(vocab, generator=g) - 4
    thread = torch.arange(vocab) // 8 % threads
    large, n = thread < 63, int((thread < 63).sum())
    z[large] = {"up": torch.linspace(20, 30, n), "down": torch.linspace(30, 20, n),
                "any": torch.linspace(20, 30, n)[torch.randperm(n, generator=g)], "one value": torch.full((n,), 25.0),
                "few values": torch.randint(20, 24, (n,), generator=g).float()}[kind]
    z[thread == 63] = 10 + torch.rand(int((thread == 63).sum()), generator=g)
    return z.to(dt)


# a row's threads: 256 up to 16384 tokens, 512 beyond, 1024 for few rows of more than 65536
@pytest.mark.parametrize("vocab,threads", [(16_000, 256), (16_383, 256), (50_257, 512), (131_077, 1024)])
@pytest.mark.parametrize("dtype", list(DT))
def test_crowded_rows(vocab, threads, dtype):
    kinds = ("up", "down", "any", "one value", "few values")
    z = torch.stack([crowded(vocab, threads, DT[dtype], k) for k in kinds])
    tokens = torch.randint(vocab, (len(kinds), 2), generator=torch.Generator().manual_seed(1))
    for top in (64, 63, 40, 8):
        run(z, tokens, top, True)
