"""The operators together, as a stack of generated linears uses them (``examples/gpt2_stack.py``)."""
import sys
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

pytestmark = pytest.mark.gpu


def make(**kw):
    from gpt2_stack import Stack

    torch.manual_seed(3)
    args = {"layers": 2, "width": 96, "heads": 3, "vocabulary": 131, "context": 80, "latent_ratio": 0.5} | kw
    return Stack(**args).cuda()


def plain(model, ids, params):
    """Logits by torch's operators in float64 on the CPU from the stack's parameters and generated weights."""
    x = F.embedding(ids, params["tokens"]) + params["positions"][: ids.shape[1]]
    batch, tokens, width = x.shape
    for i in range(len(model.blocks)):
        g = {k.split(".", 1)[1]: v for k, v in params.items() if k.startswith(f"{i}.")}
        n = F.layer_norm(x, (width,), g["n1w"], g["n1b"])
        q, k, v = (n @ g["qkv"].T).view(batch, tokens, 3, model.heads, -1).permute(2, 0, 3, 1, 4)
        s = q @ k.transpose(-1, -2) / q.shape[-1] ** 0.5
        s = s.masked_fill(torch.ones(tokens, tokens).triu(1).bool(), float("-inf"))
        x = x + (s.softmax(-1) @ v).transpose(1, 2).reshape(batch, tokens, width) @ g["proj"].T
        n = F.layer_norm(x, (width,), g["n2w"], g["n2b"])
        x = x + F.gelu(n @ g["up"].T + g["up_bias"], approximate="tanh") @ g["down"].T
    return F.layer_norm(x, (width,), params["nw"], params["nb"]) @ params["tokens"].T


def plain_params(model):
    def leaf(t):
        return t.detach().double().cpu().requires_grad_(True)

    out = {"tokens": leaf(model.tokens.weight), "positions": leaf(model.positions.weight),
           "nw": leaf(model.norm.weight), "nb": leaf(model.norm.bias)}
    for i, b in enumerate(model.blocks):
        out |= {f"{i}.n1w": leaf(b.norm1.weight), f"{i}.n1b": leaf(b.norm1.bias), f"{i}.n2w": leaf(b.norm2.weight),
                f"{i}.n2b": leaf(b.norm2.bias), f"{i}.up_bias": leaf(b.up_bias)}
        out |= {f"{i}.{k}": leaf(getattr(b, k).weight) for k in ("qkv", "proj", "up", "down")}
    return out


def rel(got, want):
    got, want = got.double().cpu(), want.double().cpu()
    return float((got - want).norm() / want.norm())


def test_step_against_plain_operators():
    import latent_weight_lab_amd as lwl

    model = make()
    ids = torch.randint(131, (3, 78), device="cuda")
    params = plain_params(model)
    want = plain(model, ids[:, :-1].cpu(), params)
    F.cross_entropy(want.flatten(0, 1), ids[:, 1:].cpu().flatten()).backward()
    lwl.prepare_block_fht_weight_cache(model)
    got = model(ids[:, :-1])
    F.cross_entropy(got.flatten(0, 1), ids[:, 1:].flatten()).backward()
    weights = {f"{i}.{k}": getattr(b, k)._cached_weight.grad
               for i, b in enumerate(model.blocks) for k in ("qkv", "proj", "up", "down")}
    # float32: some 20 operations in a row, each of a few 2^-24, and library products of up to 384 terms
    assert rel(got, want) < 1e-5
    # the checkpoint of 8 bits: its error is at most max|z| / 254 of a group of 128, some 3.5 / 254 / sqrt(3) =
    # 0.8 % of z's spread; each of the two blocks moves gelu' (slope at most 0.8) and the activation by about
    # as much, the gradients by 1 % a block, twice that allowed
    for name, grad in weights.items():
        assert rel(grad, params[name].grad) < 0.04, name
    for i, b in enumerate(model.blocks):
        assert rel(b.up_bias.grad, params[f"{i}.up_bias"].grad) < 0.04
        assert rel(b.norm1.weight.grad, params[f"{i}.n1w"].grad) < 0.04
        assert rel(b.norm2.bias.grad, params[f"{i}.n2b"].grad) < 0.04
    assert rel(model.tokens.weight.grad, params["tokens"].grad) < 0.04
    assert rel(model.positions.weight.grad[:77], params["positions"].grad[:77]) < 0.04
    lwl.flush_block_fht_weight_cache(model)
    for b in model.blocks:
        for m in (b.qkv, b.proj, b.up, b.down):
            latent = m.generator.latent
            assert latent.grad is not None and torch.isfinite(latent.grad).all() and latent.grad.abs().max() > 0


@pytest.mark.parametrize("dtype, tol", [
    (torch.float32, 1e-5),   # the same operations in another order
    (torch.bfloat16, 3e-2),  # each of some 12 roundings a block to 2^-9, of two blocks, adds up as its root: 2^-9 * 5
])
def test_decoding_is_the_whole_forward(dtype, tol):
    """Prompts of several lengths, padded, then token by token: the logits are those of the whole sequence in one
    forward pass."""
    import latent_weight_lab_amd as lwl

    model = make().to(dtype)
    lengths = torch.tensor([1, 17, 33, 40], device="cuda")
    prompts = torch.randint(131, (4, 40), device="cuda")
    tokens, logits = model.decode(prompts, lengths, 7)
    assert tokens.shape == (4, 7) and logits.shape == (4, 7, 131)
    with torch.no_grad():
        lwl.prepare_block_fht_weight_cache(model)
        for b, n in enumerate(lengths.tolist()):
            whole = torch.cat([prompts[b, :n], tokens[b]])[None]
            want = model(whole)[0, n - 1:-1]
            assert rel(logits[b], want) < tol
        lwl.flush_block_fht_weight_cache(model)


def test_training_lowers_the_loss():
    model = make(width=128, heads=2).bfloat16()
    ids = torch.randint(131, (2, 65), device="cuda")
    optimizer = torch.optim.AdamW(model.parameters(), lr=3e-3)
    losses = [float(model.step(ids[:, :-1], ids[:, 1:], optimizer)) for _ in range(20)]
    assert losses[-1] < losses[0] - 0.5, losses
