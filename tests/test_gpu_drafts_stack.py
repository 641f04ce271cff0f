"""Windows, drafted trees and tokens' log probabilities together, as a stack of generated linears uses them
(``examples/gpt2_stack.py``)."""
import pytest
import torch
import torch.nn.functional as F

from test_gpu_gpt2_stack import make, plain_params, rel

pytestmark = pytest.mark.gpu


def local_plain(model, ids, params, window, sinks):
    """Logits by torch's operators in float64 on the CPU, attention local."""
    x = F.embedding(ids, params["tokens"]) + params["positions"][: ids.shape[1]]
    batch, tokens, width = x.shape
    i = torch.arange(tokens)
    hidden = (i > i[:, None]) | ((i[:, None] - i >= window) & (i >= sinks))
    for n in range(len(model.blocks)):
        g = {k.split(".", 1)[1]: v for k, v in params.items() if k.startswith(f"{n}.")}
        y = F.layer_norm(x, (width,), g["n1w"], g["n1b"])
        q, k, v = (y @ g["qkv"].T).view(batch, tokens, 3, model.heads, -1).permute(2, 0, 3, 1, 4)
        s = (q @ k.transpose(-1, -2) / q.shape[-1] ** 0.5).masked_fill(hidden, float("-inf"))
        x = x + (s.softmax(-1) @ v).transpose(1, 2).reshape(batch, tokens, width) @ g["proj"].T
        y = F.layer_norm(x, (width,), g["n2w"], g["n2b"])
        x = x + F.gelu(y @ g["up"].T + g["up_bias"], approximate="tanh") @ g["down"].T
    return F.layer_norm(x, (width,), params["nw"], params["nb"]) @ params["tokens"].T


def test_a_local_stack_against_plain_operators():
    """Logits, the loss of next tokens, some of them padding, and gradients."""
    import latent_weight_lab_amd as lwl

    model = make(window=11, sinks=2)
    ids = torch.randint(131, (3, 78), device="cuda")
    targets = ids[:, 1:].clone()
    targets[1, 50:] = -1
    params = plain_params(model)
    want = local_plain(model, ids[:, :-1].cpu(), params, 11, 2)
    loss = F.cross_entropy(want.flatten(0, 1), targets.cpu().flatten(), ignore_index=-1, reduction="sum")
    loss.backward()
    lwl.prepare_block_fht_weight_cache(model)
    got = model(ids[:, :-1])
    ours = -lwl.token_log_probs(got, targets).sum()
    ours.backward()
    # as for the stack without a window: some 20 operations in a row, each of a few 2^-24; 227 terms of about log 131
    assert rel(got, want) < 1e-5 and abs(ours.item() - loss.item()) < 1e-4 * loss.item()
    # the activations' checkpoint of 8 bits decides, as there
    for i, b in enumerate(model.blocks):
        for k in ("qkv", "proj", "up", "down"):
            assert rel(getattr(b, k)._cached_weight.grad, params[f"{i}.{k}"].grad) < 0.04, (i, k)
    assert rel(model.tokens.weight.grad, params["tokens"].grad) < 0.04
    lwl.flush_block_fht_weight_cache(model)


@pytest.mark.parametrize("dtype, tol", [
    (torch.float32, 1e-5),   # the same operations in another order
    (torch.bfloat16, 3e-2),  # each of some 12 roundings a block to 2^-9, of two blocks, adds up as its root: 2^-9 * 5
])
def test_local_decoding_is_the_whole_forward(dtype, tol):
    import latent_weight_lab_amd as lwl

    model = make(window=9, sinks=1).to(dtype)
    lengths = torch.tensor([1, 17, 33, 40], device="cuda")
    prompts = torch.randint(131, (4, 40), device="cuda")
    tokens, logits = model.decode(prompts, lengths, 7)
    with torch.no_grad():
        lwl.prepare_block_fht_weight_cache(model)
        for b, n in enumerate(lengths.tolist()):
            whole = torch.cat([prompts[b, :n], tokens[b]])[None]
            assert rel(logits[b], model(whole)[0, n - 1:-1]) < tol
        lwl.flush_block_fht_weight_cache(model)


def oracle_drafts(answers, lengths, wrong):
    """Trees of what the model will say, three tokens ahead, beside a branch of what it will not; every node's number is
    scrambled, so that a path's keys lie apart."""
    def draft(known):
        tokens, parents = [], []
        for k, answer, n in zip(known, answers, lengths):
            ahead = answer[len(k) - n: len(k) - n + 3]
            t, p, node = [k[-1]], [-1], 0
            for step, token in enumerate(ahead):
                other = (token + 1) % 131
                t.append(other)  # a sibling first
                p.append(node)
                t.append(other if step == wrong else token)
                p.append(node if step != wrong else len(t) - 2)
                node = len(t) - 1
            t += [0] * (7 - len(t))
            p += [-1] * (7 - len(p))
            tokens.append(t)
            parents.append(p)
        return tokens, parents
    return draft


@pytest.mark.parametrize("wrong, passes", [(None, 3), (0, 9), (1, 5)])
def test_drafts_give_what_single_tokens_give(wrong, passes):
    """The greedy continuation, in fewer passes the more drafts are right, with its log probabilities."""
    model = make()
    lengths = torch.tensor([3, 17, 33, 40], device="cuda")
    prompts = torch.randint(131, (4, 40), device="cuda")
    tokens, logits = model.decode(prompts, lengths, 10)
    draft = oracle_drafts(tokens.tolist(), lengths.tolist(), wrong)
    got, log_probs, used = model.decode_drafts(prompts, lengths, 10, draft)
    assert torch.equal(got, tokens.cpu())
    # the first token comes with the prompt; a pass yields a token and what the drafts got right
    assert used == passes
    want = logits.double().log_softmax(-1).gather(-1, tokens[..., None])[..., 0].cpu()
    # float32 logits of a few units, computed in another order (1e-5 relative, above)
    assert (log_probs.double() - want).abs().max() < 1e-4


def test_drafts_from_the_sequences_themselves():
    from gpt2_stack import repeats

    model = make()
    lengths = torch.tensor([12, 40], device="cuda")
    prompts = torch.randint(5, (2, 40), device="cuda")  # few different tokens: much to draft from
    tokens, _ = model.decode(prompts, lengths, 20)
    got, _, passes = model.decode_drafts(prompts, lengths, 20, repeats)
    assert torch.equal(got, tokens.cpu()) and 1 <= passes <= 19


def test_the_step_trains():
    """The example's step runs and leaves gradients; its loss is torch's cross entropy."""
    model = make(window=20, sinks=1).bfloat16()
    ids = torch.randint(131, (2, 65), device="cuda")
    with torch.no_grad():
        want = F.cross_entropy(model(ids[:, :-1]).flatten(0, 1).double(), ids[:, 1:].flatten())
    optimizer = torch.optim.AdamW(model.parameters(), lr=1e-3)
    loss = model.step(ids[:, :-1], ids[:, 1:], optimizer)
    # the weights' cache rounds the generated weights as the uncached forward does: the same logits, some of whose sums
    # may round otherwise (2^-9 of values of a few units, averaged over 128 rows)
    assert abs(loss.item() - want.item()) < 2e-2
    for b in model.blocks:
        grad = b.qkv.generator.latent.grad
        assert grad is not None and torch.isfinite(grad).all() and grad.abs().max() > 0
