"""Layer norm (``layer_norm``, ``lwl_layer_norm_*``) against float64, forward and backward.

Bounds: y = n w + b with n computed in float32 from a mean and a variance that are off by a few
roundings each: |error| <= u |y| + 2^-19 (|n w| + |b| + |mean| s |w|), u the type's roundoff.  dx the same
with the sizes of its terms, the sums over rows 2^-18 of the sum of their terms' sizes.
"""
from __future__ import annotations

import pytest
import torch

import layer_oracle as R
from conftest import gpu_available
from latent_weight_lab_amd import LayerNorm, layer_norm
from latent_weight_lab_amd import _native as N

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5

# lanes of a wave, a wave, several waves, the last size of each kind and one past it, rows read again
SHAPES = [(1, 1), (1, 768), (3, 5), (70, 7), (33, 128), (9, 129), (8, 512), (17, 513), (2051, 768), (5, 1000),
          (64, 1024), (7, 1025), (5, 2048), (3, 3071), (4, 4096), (3, 4097), (3, 8192), (3, 8193), (2, 20001)]


def make(rows, f, dt, wt, seed, bias=True, residual=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    x = (r(rows, f) * (0.5 + r(f).abs()) + r(f)).to(dt)
    w = (1 + 0.2 * r(f)).to(wt)
    b = (0.2 * r(f)).to(wt) if bias else None
    res = r(rows, f).to(dt) if residual else None
    return x, w, b, res, r(rows, f).to(dt), r(rows, f).to(dt)


def gpu(t, grad=False):
    return None if t is None else t.cuda().requires_grad_(grad)


def check(rows, f, dt, wt, x, w, b, res, dy, dh, out, grads):
    h = x if res is None else (x.float() + res.float()).to(dt)
    u = R.U[dt]
    y, n, rstd = R.layer_norm(h, w, b, EPS)
    wd = w.double()
    size = (n * wd).abs() + (0 if b is None else b.double().abs()) + (h.double().mean(-1, keepdim=True) * rstd * wd).abs()
    if res is not None:
        assert torch.equal(out[1].cpu(), h)
    assert ((out[0].double().cpu() - y).abs() <= u * y.abs() + 2.0 ** -19 * size + R.TINY[dt]).all()
    if grads is None:
        return
    _, dx, dw, db = R.layer_norm(h, w, b, EPS, dy, dh if res is not None else None)
    a = (dy.double() * wd).abs()
    nn = n.abs() + (h.double().mean(-1, keepdim=True) * rstd).abs() * 2.0 ** -2 + 1
    size = rstd * (a + a.mean(-1, keepdim=True) + nn * (a * nn).mean(-1, keepdim=True)) + dh.double().abs()
    assert ((grads[0].double().cpu() - dx).abs() <= u * dx.abs() + 2.0 ** -18 * size + R.TINY[dt]).all()
    uw = R.U[wt]
    assert ((grads[1].double().cpu() - dw).abs() <= uw * dw.abs() + 2.0 ** -18 * (dy.double().abs() * nn).sum(0) + R.TINY[wt]).all()
    if b is not None:
        assert ((grads[2].double().cpu() - db).abs() <= uw * db.abs() + 2.0 ** -18 * dy.double().abs().sum(0) + R.TINY[wt]).all()


@pytest.mark.parametrize("rows,f", SHAPES)
@pytest.mark.parametrize("dtype,wtype", [("f32", "f32"), ("f16", "f16"), ("bf16", "f32")])
def test_step_matches_float64(rows, f, dtype, wtype):
    dt, wt = DT[dtype], DT[wtype]
    x, w, b, res, dy, dh = make(rows, f, dt, wt, rows * 7 + f)
    gx, gw, gb, gr = gpu(x, True), gpu(w, True), gpu(b, True), gpu(res, True)
    out = layer_norm(gx, gw, gb, EPS, gr)
    grads = torch.autograd.grad(out, (gx, gw, gb, gr), (dy.cuda(), dh.cuda()))
    assert torch.equal(grads[0], grads[3])
    check(rows, f, dt, wt, x, w, b, res, dy, dh, out, grads)


@pytest.mark.parametrize("rows,f", [(1, 768), (300, 96), (5, 3072), (2, 9000)])
@pytest.mark.parametrize("dtype,wtype", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
def test_plain_without_bias(rows, f, dtype, wtype):
    dt, wt = DT[dtype], DT[wtype]
    x, w, b, _, dy, dh = make(rows, f, dt, wt, 3 + f, bias=False, residual=False)
    gx, gw = gpu(x, True), gpu(w, True)
    out = layer_norm(gx, gw, eps=EPS)
    grads = torch.autograd.grad(out, (gx, gw), dy.cuda())
    with torch.no_grad():
        assert torch.equal(layer_norm(gx, gw, eps=EPS), out)
    check(rows, f, dt, wt, x, w, None, None, dy, torch.zeros_like(dh), [out], grads)


def test_layouts_and_partial_gradients():
    x, w, b, res, dy, dh = make(40, 100, torch.bfloat16, torch.float32, 1)
    want = layer_norm(x.cuda(), w.cuda(), b.cuda(), EPS, res.cuda())
    wide = torch.zeros(40, 211, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:103] = x.cuda()  # a view whose rows start at odd offsets
    got = layer_norm(wide[:, 3:103], w.cuda(), b.cuda(), EPS, res.t().contiguous().cuda().t())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    flat = torch.zeros(4001, dtype=torch.bfloat16, device="cuda")
    flat[1:] = x.reshape(-1).cuda()
    got = layer_norm(flat[1:].view(4, 10, 100), w.cuda(), b.cuda(), EPS, res.view(4, 10, 100).cuda())
    assert torch.equal(got[0].view(40, 100), want[0])
    # only the sum's gradient, only the norm's, only the weight's
    gx, gr = gpu(x, True), gpu(res, True)
    y, h = layer_norm(gx, w.cuda(), b.cuda(), EPS, gr)
    assert torch.equal(torch.autograd.grad(h, gx, dh.cuda(), retain_graph=True)[0], dh.cuda())
    alone = torch.autograd.grad(y, gx, dy.cuda(), retain_graph=True)[0]
    both = torch.autograd.grad((y, h), gx, (dy.cuda(), torch.zeros_like(dh).cuda()))[0]
    assert torch.equal(alone, both)
    gw = gpu(w, True)
    layer_norm(x.cuda(), gw, b.cuda(), EPS).backward(dy.cuda())
    assert gw.grad is not None and torch.isfinite(gw.grad).all()


def test_empty_and_constant_rows():
    w, b = torch.ones(768, device="cuda", requires_grad=True), torch.zeros(768, device="cuda", requires_grad=True)
    e = layer_norm(torch.empty(0, 768, device="cuda", requires_grad=True), w, b)
    assert e.shape == (0, 768)
    e.sum().backward()
    assert torch.equal(w.grad, torch.zeros_like(w)) and torch.equal(b.grad, torch.zeros_like(b))
    x = torch.full((5, 768), 3.0, device="cuda")  # variance 0: eps alone
    assert torch.equal(layer_norm(x, w.detach(), b.detach()), torch.zeros_like(x))
    x[2, 5] = float("nan")
    y = layer_norm(x, w.detach(), b.detach())
    assert y[2].isnan().all() and torch.equal(y[[0, 1, 3, 4]], torch.zeros(4, 768, device="cuda"))


def test_repeats_bit_for_bit_on_another_stream_and_in_a_graph():
    x, w, b, res, dy, dh = (t.cuda() for t in make(3000, 768, torch.bfloat16, torch.float32, 5))
    gx, gw, gb = x.clone().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()

    def step():
        out = layer_norm(gx, gw, gb, EPS, res)
        return list(out) + list(torch.autograd.grad(out, (gx, gw, gb), (dy, dh)))

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            got = step()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        y, h = layer_norm(x, w, b, EPS, res)
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(h, want[1])


def test_module_and_refusals():
    m = LayerNorm(64, bias=False).cuda()
    assert m.bias is None and m(torch.randn(2, 3, 64, device="cuda")).shape == (2, 3, 64)
    x = torch.randn(4, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    for bad in (lambda: layer_norm(x, w[:63]), lambda: layer_norm(x, w, w.half()), lambda: layer_norm(x, w.half()),
                lambda: layer_norm(x, w, residual=x[:3]), lambda: layer_norm(x, w, residual=x.half()),
                lambda: layer_norm(x, w, eps=-1.0), lambda: layer_norm(x, w, eps=float("nan")),
                lambda: layer_norm(x.double(), w.double()), lambda: layer_norm(x.cpu(), w.cpu()),
                lambda: layer_norm(x[:, :0], w[:0])):
        with pytest.raises((RuntimeError, ValueError)):
            bad()
    xg = x.clone().requires_grad_()
    g = torch.autograd.grad(layer_norm(xg, w).sum(), xg, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()
    assert issubclass(N.BlockFHTArgumentError, ValueError)


def test_saved_tensors_in_another_layout_or_type():
    """A caller's hooks may give saved tensors back in another layout, statistics only as they were."""
    x, w = torch.randn(30, 100, device="cuda", requires_grad=True), torch.randn(100, device="cuda", requires_grad=True)
    dy = torch.randn(30, 100, device="cuda")
    want = torch.autograd.grad(layer_norm(x, w), (x, w), dy)
    apart = lambda t: torch.stack([t, t], -1)[..., 0]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t if t.shape == (2, 30) else apart(t)):
        y = layer_norm(x, w)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (x, w), dy), want))
    for change in (apart, torch.Tensor.half, lambda t: t[:, :29].contiguous()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: change(t) if t.shape == (2, 30) else t):
            y = layer_norm(x, w)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, (x, w), dy)


@pytest.mark.parametrize("rows,f", [(1, 768), (70, 300), (3, 9000)])
@pytest.mark.parametrize("dtype,wtype", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("frozen", [False, True])
def test_residual_without_bias(rows, f, dtype, wtype, frozen):
    """The residual is the third tensor then; with x frozen its gradient is the residual's alone."""
    dt, wt = DT[dtype], DT[wtype]
    x, w, _, res, dy, dh = make(rows, f, dt, wt, rows + f, bias=False)
    gx, gw, gr = gpu(x, not frozen), gpu(w, True), gpu(res, True)
    out = layer_norm(gx, gw, None, EPS, gr)
    wanted = (gw, gr) if frozen else (gx, gw, gr)
    grads = torch.autograd.grad(out, wanted, (dy.cuda(), dh.cuda()))
    if not frozen:
        assert torch.equal(grads[0], grads[2])
    # As check()'s bounds, and the error of the mean's sum, 2^-19 of the mean size: a row whose mean is almost zero
    # and that has no bias holds nothing else to measure a small n by.
    h, u, uw = (x.float() + res.float()).to(dt), R.U[dt], R.U[wt]
    y, n, rstd = R.layer_norm(h, w, None, EPS)
    _, dx, dw, _ = R.layer_norm(h, w, None, EPS, dy, dh)
    off_mean, wd = h.double().abs().mean(-1, keepdim=True) * rstd, w.double()
    assert torch.equal(out[1].cpu(), h)
    assert ((out[0].double().cpu() - y).abs() <= u * y.abs() + 2.0 ** -19 * (n.abs() + off_mean) * wd.abs() + R.TINY[dt]).all()
    a, nn = (dy.double() * wd).abs(), n.abs() + off_mean
    size = rstd * (a + a.mean(-1, keepdim=True) + nn * (a * nn).mean(-1, keepdim=True)) + dh.double().abs()
    assert ((grads[-1].double().cpu() - dx).abs() <= u * dx.abs() + 2.0 ** -18 * size + R.TINY[dt]).all()
    assert ((grads[-2].double().cpu() - dw).abs() <= uw * dw.abs() + 2.0 ** -18 * (dy.double().abs() * nn).sum(0) + R.TINY[wt]).all()


def test_rows_that_are_not_dense_are_made_so_once():
    """The copy that the kernel reads is the one kept for the backward pass."""
    wide = torch.randn(2000, 1500, device="cuda", requires_grad=True)
    w = torch.ones(1000, device="cuda")
    layer_norm(wide[:, :1000], w)
    before = torch.cuda.memory_stats()["requested_bytes.all.allocated"]
    y = layer_norm(wide[:, :1000], w)
    asked = torch.cuda.memory_stats()["requested_bytes.all.allocated"] - before
    assert asked == 2 * 2000 * 1000 * 4 + 2 * 2000 * 4
    dy = torch.randn_like(y)
    dense = wide[:, :1000].detach().contiguous().requires_grad_()
    want = torch.autograd.grad(layer_norm(dense, w), dense, dy)[0]
    got = torch.autograd.grad(y, wide, dy)[0]
    assert torch.equal(got[:, :1000], want) and (got[:, 1000:] == 0).all()
