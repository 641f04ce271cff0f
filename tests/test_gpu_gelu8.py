"""GELU with its input kept in 8 bits (``gelu_checkpoint8``, ``lwl_gelu8_*``).

Bounds.  Value and slope: Phi's tail h = 1 - Phi(|z|) is a fit of relative error 5e-6 (16-bit outputs) or
4e-7 (float32), times exp(-z^2/2) whose argument is off by a few roundings; with the tanh form the logistic
function's argument is off by 2^-21 of itself.  The checkpoint's codes and scales are what float32 gives
by the definition, to the last bit.
"""
from __future__ import annotations

import math

import pytest
import torch

import layer_oracle as R
from conftest import gpu_available
from latent_weight_lab_amd import BlockFHTLinear, gelu_checkpoint8, gelu_linear_checkpoint8, layer_ops
from latent_weight_lab_amd import prepare_block_fht_weight_cache

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SHAPES = [(1, 1), (1, 3072), (3, 7), (130, 8), (5, 127), (9, 128), (6, 129), (33, 200), (4, 511), (7, 512), (6, 513),
          (16, 3072), (1027, 1000), (5000, 384)]


def slack(z, dt, approximate):
    """(absolute error of the value, of the slope) before the rounding to the type."""
    z = z.double()
    if approximate == "tanh":
        u2 = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        s = torch.sigmoid(u2)
        e = s * (1 - s) * (u2.abs() + 1) * 2.0 ** -20 + s * 2.0 ** -21
        grow = (1 + 2 * (z.abs() + z.abs() ** 3))
        return z.abs() * e, e * grow
    h = 0.5 * torch.erfc(z.abs() / math.sqrt(2.0))
    rel = 1.2e-6 if dt == torch.float32 else 8e-6
    rel = rel + (0 if dt == torch.float32 else 1) * z * z * 2.0 ** -22
    phi = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return z.abs() * h * rel + z.abs() * 2.0 ** -23, (h + z.abs() * phi) * rel + 2.0 ** -22


def make(rows, f, dt, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, f, generator=g) * torch.exp(torch.randn(f, generator=g))).to(dt)
    return x, (0.3 * torch.randn(f, generator=g)).to(dt), torch.randn(rows, f, generator=g).to(dt)


@pytest.mark.parametrize("rows,f", SHAPES)
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("approximate", ["none", "tanh"])
def test_step_matches_float64(rows, f, dtype, approximate):
    dt = DT[dtype]
    x, b, dy = make(rows, f, dt, rows + 13 * f)
    gx, gb = x.cuda().requires_grad_(), b.cuda().requires_grad_()
    y, kept = gelu_checkpoint8(gx, gb, approximate, return_checkpoint=True)
    z = x.float() + b.float()
    u = R.U[dt]
    want, _ = R.gelu(z, approximate)
    off = slack(z, dt, approximate)[0]
    assert ((y.detach().double().cpu() - want).abs() <= u * want.abs() + off + R.TINY[dt]).all()
    codes, scales = R.checkpoint8(z)
    assert torch.equal(kept.codes[:, :f].cpu(), codes)
    assert torch.equal(kept.scales.cpu(), scales)
    zk = (codes.float() * scales.repeat_interleave(128, 1)[:, :f])
    assert torch.equal(kept.values().cpu(), zk)
    again, slope = R.gelu(zk, approximate)
    off_v, off_s = slack(zk, dt, approximate)
    got = kept.activation()
    assert got.dtype == dt and ((got.double().cpu() - again).abs() <= u * again.abs() + off_v + R.TINY[dt]).all()
    dx, db = torch.autograd.grad(y, (gx, gb), dy.cuda())
    d = dy.double()
    assert ((dx.double().cpu() - d * slope).abs() <= u * (d * slope).abs() + d.abs() * off_s + R.TINY[dt]).all()
    want_b = (d * slope).sum(0)
    off_b = (d.abs() * (off_s + slope.abs() * 2.0 ** -18)).sum(0)
    assert ((db.double().cpu() - want_b).abs() <= u * want_b.abs() + off_b + R.TINY[dt]).all()
    with torch.no_grad():
        assert torch.equal(gelu_checkpoint8(gx, gb, approximate), y)


def test_extremes():
    for dt in DT.values():
        big = 6e4 if dt == torch.float16 else 1e30
        x = torch.zeros(6, 256, dtype=dt)
        x[0, :4] = torch.tensor([big, -big, 1.0, -1.0])
        x[1, 5] = float("inf")
        x[2, 6] = float("-inf")
        x[3, 7] = float("nan")
        x[5] = 1e-7
        y, kept = gelu_checkpoint8(x.cuda(), return_checkpoint=True)
        y, v = y.float().cpu(), kept.values().cpu()
        assert y[0, 0] == x[0, 0].float() and y[0, 1] == 0
        assert y[1, 5] == float("inf") and y[2, 6] == 0 and y[3, 7].isnan()
        for row in (1, 2, 3):  # the group that went wrong shows it, the other does not
            assert v[row, :128].isnan().all() and (v[row, 128:] == 0).all()
        assert (v[4] == 0).all() and (y[4] == 0).all()
        if dt != torch.float16:
            assert torch.allclose(v[5], x[5].float(), rtol=1 / 127)
        g, _ = layer_ops.gelu8_backward(kept.codes, kept.scales, torch.ones(6, 256, dtype=dt, device="cuda"), dt, "none", False)
        assert g[1, :128].isnan().all() and torch.isfinite(g[0]).all() and g[0, 0] == 1 and g[0, 1] == 0
        t = gelu_checkpoint8(x.cuda(), approximate="tanh").float().cpu()
        assert t[0, 0] == x[0, 0].float() and t[0, 1] == 0 and t[1, 5] == float("inf") and t[2, 6] == 0 and t[3, 7].isnan()
    tiny = torch.full((1, 128), 1e-38)
    _, kept = gelu_checkpoint8(tiny.cuda(), return_checkpoint=True)
    assert (kept.values() == 0).all()


def test_layouts_streams_and_graph():
    x, b, dy = make(300, 513, torch.bfloat16, 3)
    want = gelu_checkpoint8(x.cuda(), b.cuda())
    wide = torch.zeros(300, 600, dtype=torch.bfloat16, device="cuda")
    wide[:, 1:514] = x.cuda()
    assert torch.equal(gelu_checkpoint8(wide[:, 1:514], b.cuda()), want)
    odd = torch.zeros(300 * 513 + 1, dtype=torch.bfloat16, device="cuda")
    odd[1:] = x.reshape(-1).cuda()
    assert torch.equal(gelu_checkpoint8(odd[1:].view(3, 100, 513), b.cuda()).view(300, 513), want)
    assert gelu_checkpoint8(x[:0].cuda(), b.cuda()).shape == (0, 513)
    gx, gb = x.cuda().requires_grad_(), b.cuda().requires_grad_()

    def step():
        return torch.autograd.grad(gelu_checkpoint8(gx, gb), (gx, gb), dy.cuda())

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    graph = torch.cuda.CUDAGraph()
    sx, sb, sd = x.cuda(), b.cuda(), dy.cuda()
    with torch.no_grad(), torch.cuda.graph(graph):
        y, kept = gelu_checkpoint8(sx, sb, return_checkpoint=True)
        dx, db = layer_ops.gelu8_backward(kept.codes, kept.scales, sd, torch.bfloat16, "none", True)
    for _ in range(3):
        y.zero_(), dx.zero_(), db.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(dx, first[0]) and torch.equal(db, first[1])


@pytest.mark.parametrize("cached", [False, True])
def test_linear_takes_its_input_from_the_checkpoint(cached):
    """The latent's gradient is that of the checkpoint's activation, and the activation is not kept."""
    torch.manual_seed(0)
    lin = BlockFHTLinear(256, 96, latent_dim=512, seed=4).cuda()
    x = torch.randn(2, 50, 256, device="cuda", requires_grad=True)
    dy = torch.randn(2, 50, 96, device="cuda")
    if cached:
        prepare_block_fht_weight_cache(lin)
    held = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: held.append(tuple(t.shape)) or t, lambda t: t):
        y = gelu_linear_checkpoint8(x, lin)
    assert not any(math.prod(s) == 2 * 50 * 256 and s[-1] == 256 for s in held if len(s) == 3)
    y.backward(dy)
    p = lin._cached_weight if cached else lin.generator.latent
    got_w, got_x = p.grad.clone(), x.grad.clone()
    p.grad = x.grad = None
    z, kept = gelu_checkpoint8(x, return_checkpoint=True)
    assert torch.equal(y, lin(z))
    lin(kept.activation()).backward(dy)
    assert torch.equal(got_w, p.grad)
    a = z.detach().requires_grad_()
    lin(a).backward(dy)
    want_x, _ = layer_ops.gelu8_backward(kept.codes, kept.scales, a.grad, x.dtype, "none", False)
    assert torch.equal(got_x, want_x)
    with torch.no_grad():
        assert torch.equal(gelu_linear_checkpoint8(x, lin), y)


def test_refusals():
    x = torch.randn(4, 64, device="cuda")
    for bad in (lambda: gelu_checkpoint8(x.double()), lambda: gelu_checkpoint8(x.cpu()),
                lambda: gelu_checkpoint8(x, x[0, :63]), lambda: gelu_checkpoint8(x, x[0].half()),
                lambda: gelu_checkpoint8(x, approximate="sigmoid"), lambda: gelu_checkpoint8(x[:, :0])):
        with pytest.raises((RuntimeError, ValueError)):
            bad()


@pytest.mark.parametrize("cached", [False, True])
@pytest.mark.parametrize("first", [torch.nn.Hardtanh, torch.nn.ReLU])
def test_module_that_changes_its_input_in_place(cached, first):
    """The gradients are those of the input that the linear saw, bit for bit.  Not in place, the linear's input is
    a tensor of its own and kept; what the first module saves may be the activation and stand for the checkpoint's."""
    torch.manual_seed(0)
    lin = BlockFHTLinear(256, 96, latent_dim=512, seed=4).cuda()
    x = torch.randn(2, 50, 256, device="cuda", requires_grad=True)
    dy = torch.randn(2, 50, 96, device="cuda")
    if cached:
        prepare_block_fht_weight_cache(lin)
    p = lin._cached_weight if cached else lin.generator.latent
    apart = first()(gelu_checkpoint8(x))
    want = torch.autograd.grad(lin(apart), (p, x), dy)
    got = torch.autograd.grad(gelu_linear_checkpoint8(x, torch.nn.Sequential(first(inplace=True), lin)), (p, x), dy)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = torch.autograd.grad(gelu_linear_checkpoint8(x, torch.nn.Sequential(first(), lin)), p, dy)
    assert torch.equal(got[0], want[0])


def test_checkpoints_that_do_not_fit_are_refused():
    """Codes and scales of another shape, type or layout than the call's would be read out of range."""
    x = torch.randn(40, 300, device="cuda")
    _, kept = gelu_checkpoint8(x, return_checkpoint=True)
    c, s = kept.codes, kept.scales
    assert c.shape == (40, 304) and s.shape == (40, 3)
    wide, tall = torch.zeros(40, 8, device="cuda"), torch.zeros(80, 304, dtype=torch.int8, device="cuda")
    for codes, scales in [(c, s[:, :2]), (c, s[:, :2].contiguous()), (c, s[:39]), (c, s.half()), (c, s.double()), (c, wide[:, :3]),
                          (c[:39], s), (c[:, :296].contiguous(), s), (c.float(), s), (c.to(torch.uint8), s), (tall[::2], s),
                          (c.view(-1), s), (c, s.view(-1)), (c, s.t().contiguous().t()), (c.cpu(), s), (c, s.cpu())]:
        with pytest.raises(RuntimeError):
            layer_ops.gelu8_activation(codes, scales, (40, 300), x.dtype, "none")
        with pytest.raises(RuntimeError):
            layer_ops.gelu8_backward(codes, scales, x, x.dtype, "none", True)
    for shape in [(40, 305), (41, 300), (40, 0), ()]:
        with pytest.raises(RuntimeError):
            layer_ops.gelu8_activation(c, s, shape, x.dtype, "none")
        with pytest.raises(RuntimeError):
            layer_ops.gelu8_backward(c, s, torch.ones(shape, device="cuda"), x.dtype, "none", True)
    kept.scales = s.bfloat16()
    with pytest.raises(ValueError):
        kept.activation()
    assert torch.equal(layer_ops.gelu8_activation(c, s, (2, 20, 300), x.dtype, "none").view(40, 300),
                       layer_ops.gelu8_activation(c, s, (40, 300), x.dtype, "none"))


@pytest.mark.parametrize("kind", ["torch", "generated", "cached"])
def test_activation_is_not_held(kind):
    """What a step holds for its backward pass, in bytes asked of the allocator: codes, scales and the result.  The
    same linear on the activation holds that as well."""
    rows, f, out = 2000, 1024, 8
    lin = torch.nn.Linear(f, out, device="cuda") if kind == "torch" else BlockFHTLinear(f, out, latent_dim=512, seed=4).cuda()
    if kind == "cached":
        prepare_block_fht_weight_cache(lin)
    x = torch.randn(2, rows // 2, f, device="cuda", requires_grad=True)
    asked = lambda: torch.cuda.memory_stats()["requested_bytes.all.current"]

    def held(step):
        step()  # library workspaces
        before = asked()
        y = step()
        return asked() - before, y

    kept = rows * f + rows * (f // 128) * 4 + rows * out * 4
    got, _ = held(lambda: gelu_linear_checkpoint8(x, lin))
    assert kept <= got < kept + 100_000
    got, _ = held(lambda: lin(gelu_checkpoint8(x)))
    assert kept + rows * f * 4 <= got < kept + rows * f * 4 + 100_000
