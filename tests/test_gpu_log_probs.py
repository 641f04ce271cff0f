"""Log probabilities of tokens (``token_log_probs``, ``lwl_log_probs_*``) against float64, both directions.  The bounds
are those of ``token_oracle.log_probs``."""
from __future__ import annotations

import math

import pytest
import torch

import token_oracle as R
from conftest import gpu_available
from latent_weight_lab_amd import token_log_probs

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def make(rows, vocab, each, dt, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(rows, vocab, generator=g) * spread).to(dt)
    return z, torch.randint(vocab, (rows, each), generator=g), g


def close(got, res, name, dt=torch.float32):
    want, bound = res[name], R.rounded_bound(res, name, dt)
    got = got.double().cpu().reshape(want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    off = (got - want).abs()
    assert (same | (off <= bound)).all(), (name, (off / bound)[~same].max().item())


def run(z, tokens, top=0, entropy=True, g=None, gh=None, gtop=None):
    """Forward and, with gradients given, backward of z as it lies on the GPU; checks both."""
    dt, rows = z.dtype, z.shape[0]
    res = R.log_probs(z.cpu(), tokens, g, gh, gtop, top)
    step = not (g is None and gh is None and gtop is None)
    leaf = z.cuda().requires_grad_(step) if not z.is_cuda else z.detach().requires_grad_(step)
    out = token_log_probs(leaf, tokens.cuda(), entropy=entropy, top=top)
    out = list(out) if isinstance(out, tuple) else [out]
    assert len(out) == 1 + entropy + 2 * (top > 0)
    close(out[0], res, "log_probs")
    if entropy:
        close(out[1], res, "entropy")
    if top:
        assert torch.equal(out[-1].cpu(), res["top_tokens"])
        close(out[-2], res, "top_log_probs")
    if step:
        pairs = [(o, s) for o, s in zip(out, [g] + ([gh] if entropy else []) + ([gtop] if top else [])) if s is not None]
        (dz,) = torch.autograd.grad([o for o, _ in pairs], [leaf], [s.cuda() for _, s in pairs])
        assert dz.dtype == dt and dz.is_contiguous()
        close(dz, res, "grad", dt)
        assert torch.isfinite(dz).all()
    return out


# a vocabulary of one, a chunk and its neighbours, a workgroup's round, several, more than one backward range
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,vocab,each,top", [(1, 1, 1, 1), (3, 7, 1, 7), (2, 8, 2, 3), (5, 9, 1, 0), (4, 255, 3, 64),
                                                 (2, 2049, 64, 1), (3, 8193, 1, 5), (7, 16_385, 4, 20), (2, 50_257, 1, 33),
                                                 (300, 130, 1, 2), (1, 131_077, 2, 64)])
def test_step_matches_float64(dtype, rows, vocab, each, top):
    z, tokens, gen = make(rows, vocab, each, DT[dtype], rows + vocab)
    grads = (torch.randn(rows, each, generator=gen), torch.randn(rows, generator=gen),
             torch.randn(rows, top, generator=gen) if top else None)
    run(z, tokens, top, True, *grads)
    run(z, tokens, 0, False, grads[0])
    run(z, tokens, top, False)
    run(z, tokens, top, True, None, grads[1], None)
    if top:
        run(z, tokens, top, True, None, None, grads[2])


@pytest.mark.parametrize("dtype", list(DT))
def test_orders_of_a_row(dtype):
    """Rows whose largest values lie together, equal values, both zeros, one value, huge and tiny spreads."""
    dt, vocab = DT[dtype], 20_011
    g = torch.Generator().manual_seed(3)
    up = torch.linspace(-8, 8, vocab)
    many = torch.full((vocab,), -4.0)
    many[torch.randperm(vocab, generator=g)[:3000]] = 2.0
    zeros = torch.zeros(vocab)
    zeros[::2] = -0.0
    together = torch.randn(vocab, generator=g)
    together[8192:8200] += 30
    one_thread = torch.randn(vocab, generator=g)  # the largest values all in one thread's part
    for c in range(3, (vocab + 7) // 8 - 1, 256):
        one_thread[c * 8:c * 8 + 8] = 20 + torch.rand(8, generator=g)
    rows = [up, up.flip(0), torch.full((vocab,), 1.5), zeros, many, together, one_thread, torch.randn(vocab, generator=g) * 1e-3,
            torch.randn(vocab, generator=g) * 1e3, -60000.0 + torch.rand(vocab, generator=g)]
    z = torch.stack(rows).to(dt)
    tokens = torch.randint(vocab, (len(rows), 3), generator=g)
    grads = torch.randn(len(rows), 3, generator=g), torch.randn(len(rows), generator=g)
    for top in (1, 8, 64):
        run(z, tokens, top, True, *grads)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("top", [0, 1, 40])
def test_masked_tokens(dtype, top):
    """Minus infinity and the type's lowest value as masks: some tokens, all but few, all but one, all."""
    dt, vocab = DT[dtype], 5003
    z, tokens, g = make(7, vocab, 2, dt, 11)
    low = torch.finfo(dt).min
    z[0, 17:4000] = -math.inf
    z[1] = -math.inf
    z[1, [5, 4999, 300]] = torch.tensor([1.0, 2.0, 2.0]).to(dt)
    z[2] = -math.inf
    z[2, 77] = -3.0
    z[3] = -math.inf
    z[4] = low
    z[5, 1:] = low
    z[6, 100:] = low
    tokens[:, 0] = torch.tensor([20, 5, 77, 9, 3, 0, 50])
    grads = torch.randn(7, 2, generator=g), torch.randn(7, generator=g)
    gtop = torch.randn(7, top, generator=g) if top else None
    out = run(z, tokens, top, True, *grads, gtop)
    assert out[0][0, 0] == -math.inf and (out[0][3] == -math.inf).all() and out[1][3] == 0.0 and out[1][2] == 0.0
    assert abs(out[1][4].item() - math.log(vocab)) < 1e-5


@pytest.mark.parametrize("dtype", list(DT))
def test_not_finite(dtype):
    """A NaN or plus infinity makes its own row NaN, and no other's."""
    z, tokens, g = make(6, 3001, 2, DT[dtype], 5)
    clean = token_log_probs(z.cuda(), tokens.cuda(), entropy=True, top=5)
    bad = z.clone()
    bad[1, 2999] = math.nan
    bad[3, 0] = math.inf
    bad[4] = math.nan
    leaf = bad.cuda().requires_grad_()
    out = token_log_probs(leaf, tokens.cuda(), entropy=True, top=5)
    rows = torch.tensor([1, 3, 4])
    keep = torch.tensor([0, 2, 5])
    for a, b in zip(out, clean):
        assert torch.equal(a[keep], b[keep])
    for t in out[:3]:
        assert t[rows].isnan().all()
    assert ((out[3] >= 0) & (out[3] < 3001)).all()
    (dz,) = torch.autograd.grad(out[0].sum() + out[1].sum(), leaf)
    assert dz[rows].isnan().any(1).all() and torch.isfinite(dz[keep]).all()


def test_tokens_none_past_and_again():
    """Padding, tokens past the vocabulary, the same token several times, among the alternatives too."""
    z, tokens, g = make(5, 1003, 6, torch.float32, 8)
    tokens[0] = -1
    tokens[1, 2:] = torch.tensor([1003, 1 << 40, -7, -(1 << 40)])
    tokens[2] = 500
    tokens[3] = z[3].argmax()
    grads = torch.randn(5, 6, generator=g), torch.randn(5, generator=g), torch.randn(5, 3, generator=g)
    out = run(z, tokens, 3, True, *grads)
    assert (out[0][0] == 0).all() and out[0][1, 2:4].isnan().all() and (out[0][1, 4:] == 0).all()
    bad = tokens.clone()
    bad[4] = 1 << 33
    leaf = z.cuda().requires_grad_()
    (dz,) = torch.autograd.grad(token_log_probs(leaf, bad.cuda()), leaf, grads[0].cuda())
    assert (dz[4] == 0).all() and torch.isfinite(dz).all()


@pytest.mark.parametrize("dtype", list(DT))
def test_layouts(dtype):
    """Shifted, padded, expanded, permuted and odd rows give what dense ones give, bit for bit."""
    dt = DT[dtype]
    g = torch.Generator().manual_seed(2)
    base = (torch.randn(4, 6, 517, generator=g) * 2).to(dt).cuda()
    tokens = torch.randint(500, (4, 5), generator=g).cuda()

    def both(view, tokens):
        leaf = view.detach().requires_grad_()
        dense = view.contiguous().detach().requires_grad_()
        a, b = (token_log_probs(t, tokens, entropy=True, top=4) for t in (leaf, dense))
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        up = [torch.ones_like(a[0]), torch.ones_like(a[1])]
        ga, gb = (torch.autograd.grad(list(o[:2]), t, up)[0] for o, t in ((a, leaf), (b, dense)))
        assert torch.equal(ga, gb) and ga.shape == view.shape

    both(base[:, :-1], tokens)                                   # the next token's
    both(base[:, 1:, 3:503], tokens)                             # and of a part of the vocabulary
    both(base.transpose(0, 1)[:5], tokens.t().contiguous())      # axes exchanged
    both(base[:, ::2, :], tokens[:, :3])
    both(base[:1].expand(4, -1, -1)[:, :5], tokens)              # shared rows
    both(base.transpose(1, 2)[:, :500], torch.randint(6, (4, 500), generator=g).cuda())  # values apart
    both(base.view(2, 2, 6, 517)[:, :, :5].permute(1, 2, 0, 3), torch.randint(517, (2, 5, 2), generator=g).cuda())
    both(base[0, 0], tokens[0, 0])                               # one row
    # every type of integers
    want = token_log_probs(base[:, :-1], tokens)
    for t in (torch.int32, torch.int16):
        assert torch.equal(token_log_probs(base[:, :-1], tokens.to(t)), want)
    assert token_log_probs(base, torch.zeros(4, 6, 0, dtype=torch.long, device="cuda")).shape == (4, 6, 0)


def test_no_tokens_asked_about():
    """Entropies and alternatives alone, with their gradients."""
    z, _, g = make(6, 2500, 1, torch.float32, 14)
    none = torch.zeros(6, 0, dtype=torch.long)
    run(z, none, 3, True, None, torch.randn(6, generator=g), torch.randn(6, 3, generator=g))


def test_two_streams_at_once():
    xs = [torch.randn(64, 30_000, device="cuda").bfloat16() for _ in range(2)]
    toks = torch.randint(30_000, (64,), device="cuda")
    want = [token_log_probs(x, toks, entropy=True, top=4) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(token_log_probs(x, toks, entropy=True, top=4))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for w, o in zip(want, got) for a, b in zip(w, o))


def test_nothing_around_a_row_counts():
    z, tokens, _ = make(9, 1001, 1, torch.bfloat16, 4)
    buf = torch.full((11, 1040), math.nan, dtype=torch.bfloat16, device="cuda")
    buf[1:10, 5:1006] = z.cuda()
    a = token_log_probs(buf[1:10, 5:1006], tokens.cuda(), entropy=True, top=9)
    b = token_log_probs(z.cuda(), tokens.cuda(), entropy=True, top=9)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_rows_past_32_bits():
    """Rows more than 2^32 bytes apart."""
    buf = torch.zeros((1 << 31) + 4096, dtype=torch.float16, device="cuda")
    z = buf.as_strided((3, 1000), ((1 << 30) + 7, 1))
    src, tokens, _ = make(3, 1000, 1, torch.float16, 6)
    z.copy_(src)
    a = token_log_probs(z, tokens.cuda(), entropy=True, top=2)
    b = token_log_probs(src.cuda(), tokens.cuda(), entropy=True, top=2)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_gradient_matches_differences():
    z, tokens, g = make(2, 41, 3, torch.float32, 9, spread=1.0)
    w = [torch.randn(2, 3, generator=g), torch.randn(2, generator=g), torch.randn(2, 4, generator=g)]

    def f(x):
        res = R.log_probs(x, tokens, top=4)
        return sum((res[n] * k).sum() for n, k in zip(("log_probs", "entropy", "top_log_probs"), w))

    leaf = z.cuda().requires_grad_()
    out = token_log_probs(leaf, tokens.cuda(), entropy=True, top=4)
    (dz,) = torch.autograd.grad([out[0], out[1], out[2]], leaf, [k.cuda() for k in w])
    for _ in range(5):
        step = torch.randn(2, 41, generator=g).double()
        diff = (f(z.double() + 1e-5 * step) - f(z.double() - 1e-5 * step)) / 2e-5
        assert abs(diff - (dz.double().cpu() * step).sum()) < 1e-4


def test_repeats_streams_and_graph():
    z, tokens, g = make(37, 9001, 2, torch.bfloat16, 12)
    leaf, toks, up = z.cuda().requires_grad_(), tokens.cuda(), torch.randn(37, 2, generator=g).cuda()

    def step():
        out = token_log_probs(leaf, toks, entropy=True, top=7)
        return [*out, torch.autograd.grad([out[0], out[1]], leaf, [up, up[:, 0]])[0]]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    # choosing tokens in a graph, two graphs in turn
    graphs, outs, ins = [], [], []
    for _ in range(2):
        x = torch.empty_like(z, device="cuda")
        x.copy_(z)
        token_log_probs(x, toks, entropy=True, top=7)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(token_log_probs(x, toks, entropy=True, top=7))
        graphs.append(graph)
        ins.append(x)
    for n in range(4):
        for graph, out, x in zip(graphs, outs, ins):
            x.copy_(torch.randn(37, 9001, generator=g))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, token_log_probs(x, toks, entropy=True, top=7)))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_every_run_gives_the_same_bits(dtype):
    """Which thread finds an alternative varies from run to run."""
    z, tokens, g = make(300, 50_257, 4, DT[dtype], 21)
    leaf, toks, up = z.cuda().requires_grad_(), tokens.cuda(), torch.randn(300, 4, generator=g).cuda()
    want = None
    for _ in range(20):
        out = token_log_probs(leaf, toks, entropy=True, top=7)
        got = [*out, torch.autograd.grad([out[0], out[1]], leaf, [up, up[:, 0]])[0]]
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_partial_use_and_second_derivatives():
    z, tokens, _ = make(4, 300, 1, torch.float32, 1)
    leaf = z.cuda().requires_grad_()
    lp, h, top, idx = token_log_probs(leaf, tokens[:, 0].cuda(), entropy=True, top=3)
    assert lp.shape == (4,) and not idx.requires_grad
    (a,) = torch.autograd.grad(h.sum(), leaf, retain_graph=True)
    (b,) = torch.autograd.grad(lp.sum(), leaf, retain_graph=True)
    (c,) = torch.autograd.grad(lp.sum() + h.sum(), leaf, retain_graph=True)
    assert (a + b - c).abs().max() < 1e-6
    (d,) = torch.autograd.grad(lp.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        d.sum().backward()
    with torch.no_grad():
        assert not token_log_probs(leaf, tokens[:, 0].cuda()).requires_grad
    # the loss as torch's
    loss = -token_log_probs(leaf, tokens[:, 0].cuda()).mean()
    want = torch.nn.functional.cross_entropy(z.double(), tokens[:, 0])
    assert abs(loss.item() - want.item()) < 1e-5


def test_refusals():
    z = torch.randn(4, 100, device="cuda")
    t = torch.zeros(4, dtype=torch.long, device="cuda")
    for bad in (lambda: token_log_probs(z, t[:3]), lambda: token_log_probs(z, t.float()), lambda: token_log_probs(z, t.bool()),
                lambda: token_log_probs(z, t[None]), lambda: token_log_probs(z, t, top=101), lambda: token_log_probs(z, t, top=-1),
                lambda: token_log_probs(torch.randn(4, 200, device="cuda"), t, top=65),
                lambda: token_log_probs(z, t[:, None].expand(4, 65)), lambda: token_log_probs(z.double(), t),
                lambda: token_log_probs(z.cpu(), t.cpu()), lambda: token_log_probs(z, t.cpu()),
                lambda: token_log_probs(z[:, :0], t), lambda: token_log_probs(z[0, 0], t[0])):
        with pytest.raises((RuntimeError, ValueError)):
            bad()
    out = token_log_probs(z[:0], t[:0], entropy=True, top=3)
    assert [tuple(o.shape) for o in out] == [(0,), (0,), (0, 3), (0, 3)]
    leaf = z[:0].detach().requires_grad_()
    (g,) = torch.autograd.grad(token_log_probs(leaf, t[:0]).sum(), leaf)
    assert g.shape == (0, 100)
