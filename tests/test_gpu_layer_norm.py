"""Layer norm against its definition in 64 bits.

Bounds, elementwise, with u half a step of the data's type and f = 2^-24.  Sums of d terms are trees of at most 32 terms
one behind another and 10 levels, or long rows of d / 1024 terms per thread: c = (42 + d / 1024) f bounds their relative error
against the sum of magnitudes.
  mean       |dmu| <= (c + f) mean|x|                centred value: e0 = |dmu| + f |x - mu|
  variance   relative c + 2 e1, with e1 = rms(e0) / sd, so 1 / sd has the relative error r = c + e1 + 4 f
  y          u |y| + |w| (e0 / sd + r |xh|) + 3 f (|xh w| + |b|)
  dx         u |dx| + [ (r + 4 f) |inner| + |xh| err(mean(g xh)) + exh |mean(g xh)| + err(mean g) + 2 f |g| ] / sd,
             with exh = e0 / sd + r |xh| + f |xh|, err(mean g) = c mean|g|, err(mean(g xh)) = c mean|g xh| + mean(|g| exh)
  dw, db     u' |dw| + (n-sum: cn = (n / 100 + 300) f) sum|dy xh| + sum(|dy| exh)
"""
import pytest
import torch

from falkon_b200.mmv_ops import layer_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"
F = 2.0**-24


def reference(x, w, b, eps, dy):
    d = x.shape[-1]
    n = x.numel() // d
    X, G0 = x.detach().double(), dy.double()
    W = torch.ones(d, device=DEV, dtype=torch.float64) if w is None else w.detach().double()
    B = torch.zeros(d, device=DEV, dtype=torch.float64) if b is None else b.detach().double()
    u, c, cn = torch.finfo(x.dtype).eps / 2, (42 + d / 1024) * F, (n / 100 + 300) * F
    up = F if w is None else torch.finfo(w.dtype).eps / 2
    mu = X.mean(-1, keepdim=True)
    C = X - mu
    sd = (C.square().mean(-1, keepdim=True) + eps).sqrt()
    xh = C / sd
    e0 = (c + F) * X.abs().mean(-1, keepdim=True) + F * C.abs()
    r = c + e0.square().mean(-1, keepdim=True).sqrt() / sd + 4 * F
    exh = e0 / sd + (r + F) * xh.abs()
    y = xh * W + B
    out = {"y": (y, u * y.abs() + W.abs() * exh + 3 * F * ((xh * W).abs() + B.abs()))}
    g = G0 * W
    m1, m2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    e1, e2 = c * g.abs().mean(-1, keepdim=True), c * (g * xh).abs().mean(-1, keepdim=True) + (g.abs() * exh).mean(-1, keepdim=True)
    inner = g - m1 - xh * m2
    dx = inner / sd
    out["dx"] = (dx, u * dx.abs() + ((r + 4 * F) * (g.abs() + m1.abs() + (xh * m2).abs()) + xh.abs() * e2 + exh * m2.abs() + e1) / sd)
    dims = tuple(range(x.dim() - 1))
    dw, db = (G0 * xh).sum(dims), G0.sum(dims)
    out["dw"] = (dw, up * dw.abs() + cn * (G0 * xh).abs().sum(dims) + (G0.abs() * exh).sum(dims))
    out["db"] = (db, up * db.abs() + cn * G0.abs().sum(dims))
    return out


def check(name, got, ref):
    want, bound = ref[name]
    assert got.shape == want.shape
    off = (got.double() - want).abs() - bound - 2.0**-24 * (got.dtype == torch.float16) - 1e-30
    assert not bool((off > 0).any()) and bool(got.isfinite().all()), f"{name}: {int((off > 0).sum())} of {off.numel()} out of bounds"


def run_and_check(x, w, b, dy, eps=1e-5):
    ref = reference(x, w, b, eps, dy)
    check("y", layer_norm(x, w, b, eps), ref)
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    it = iter(leaves)
    args = [None if t is None else next(it) for t in (x, w, b)]
    y = layer_norm(*args, eps)
    grads = torch.autograd.grad(y, leaves, dy)
    check("y", y.detach(), ref)
    names = [n for n, t in zip(("dx", "dw", "db"), (x, w, b)) if t is not None]
    for n, g, leaf in zip(names, grads, leaves):
        assert g.dtype == leaf.dtype
        check(n, g, ref)
    again = torch.autograd.grad(layer_norm(*args, eps), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))


def make(shape, dtype, wdtype, seed=0, weights=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(shape, device=DEV, generator=g) * 2 + 0.5
    dy = torch.randn(shape, device=DEV, generator=g)
    w = 1 + 0.3 * torch.randn(shape[-1], device=DEV, generator=g)
    b = 0.3 * torch.randn(shape[-1], device=DEV, generator=g)
    return x.to(dtype), w.to(wdtype) if weights else None, b.to(wdtype) if weights else None, dy.to(dtype)


TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)]


@pytest.mark.parametrize("dtype,wdtype", TYPES)
@pytest.mark.parametrize("rows", [1, 3, 700])
@pytest.mark.parametrize("d", [1, 2, 7, 8, 33, 64, 128, 257, 1000, 1537, 2048, 4100, 8192])
def test_sizes(d, rows, dtype, wdtype):
    run_and_check(*make((rows, d), dtype, wdtype))


@pytest.mark.parametrize("dtype,wdtype", TYPES)
@pytest.mark.parametrize("d", [12288, 16001, 16384, 40000, 65536])
def test_long_rows(d, dtype, wdtype):
    run_and_check(*make((5, d), dtype, wdtype))


@pytest.mark.parametrize("dtype,wdtype", TYPES)
@pytest.mark.parametrize("d", [8, 100, 1024])
def test_many_rows(d, dtype, wdtype):
    run_and_check(*make((20011, d), dtype, wdtype))


@pytest.mark.parametrize("which", [(False, False), (True, False), (False, True)])
def test_without_weight_or_bias(which):
    x, w, b, dy = make((50, 96), torch.bfloat16, torch.float32)
    run_and_check(x, w if which[0] else None, b if which[1] else None, dy)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_rows(dtype):
    x, w, b, dy = make((4, 30, 10, 64), dtype, torch.float32)
    for view in (x[:, :, 2:7], x[:, ::2], x[:, :, :, 8:40], x[:, :, :, 3:36], x.transpose(1, 2), x[0], x[:1, :1, 3], x.transpose(2, 3), x[1:, 3:, 1:, :17],
                 x[:, :, :1].expand(4, 30, 5, 64)):
        d = view.shape[-1]
        g = torch.randn(view.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(dtype)
        ww = 1 + 0.1 * torch.arange(d, device=DEV, dtype=torch.float32) / d
        run_and_check(view, ww, -ww, g)
    x0, w0 = x.detach().requires_grad_(), w.detach().requires_grad_()
    layer_norm(x0, w0, None).sum().backward()  # a broadcast upstream gradient
    ref = reference(x, w, None, 1e-5, torch.ones_like(x))
    check("dx", x0.grad, ref)
    check("dw", w0.grad, ref)


def test_large_mean():
    """A mean a thousand times the spread: the variance comes from centred values and keeps its digits."""
    x, w, b, dy = make((64, 777), torch.float32, torch.float32)
    run_and_check(x + 2000.0, w, b, dy)


def test_constant_rows():
    x, w, b, dy = make((4, 64), torch.float32, torch.float32)
    x = torch.full_like(x, 3.0)
    assert torch.equal(layer_norm(x, w, b), b.expand(4, 64))


@pytest.mark.parametrize("shape", [(0, 16), (3, 0, 16)])
def test_no_rows(shape):
    x = torch.empty(shape, device=DEV, requires_grad=True)
    w, b = torch.ones(16, device=DEV, requires_grad=True), torch.zeros(16, device=DEV, requires_grad=True)
    y = layer_norm(x, w, b)
    assert y.shape == x.shape
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert dx.shape == x.shape and bool((dw == 0).all()) and bool((db == 0).all())


def test_only_some_gradients():
    x, w, b, dy = make((300, 200), torch.float32, torch.float32)
    ref = reference(x, w, b, 1e-5, dy)
    for name, at in (("dx", 0), ("dw", 1), ("db", 2)):
        ts = [t.detach().requires_grad_(i == at) for i, t in enumerate((x, w, b))]
        check(name, torch.autograd.grad(layer_norm(*ts), ts[at], dy)[0], ref)


def test_other_stream_and_graph():
    x, w, b, dy = make((513, 384), torch.bfloat16, torch.float32)
    x, w, b = (t.detach().requires_grad_() for t in (x, w, b))
    want = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)
    for g in got:
        g.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_gradients_against_differences():
    x, w, b, dy = make((3, 9), torch.float32, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    h = 2.0**-8  # central differences in 64 bits: their error is h^2 f''' / 6, below 1e-4 here
    for which, g in enumerate(grads):
        for at in range(g.numel()):
            ends = []
            for sign in (1, -1):
                moved = [t.detach().double() for t in (x, w, b)]
                moved[which] = moved[which].clone()
                moved[which].view(-1)[at] += sign * h
                X, W, B = moved
                C = X - X.mean(-1, keepdim=True)
                y = C / (C.square().mean(-1, keepdim=True) + 1e-5).sqrt() * W + B
                ends.append(float((y * dy.double()).sum()))
            assert abs((ends[0] - ends[1]) / (2 * h) - float(g.reshape(-1)[at])) < 1e-3
