"""Layer norm where the data's values, not its layout, make it hard."""
import pytest
import torch

from falkon_b200.mmv_ops import layer_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"
F = 2.0**-24


@pytest.mark.parametrize("d", [777, 16384, 16385, 1 << 18, 1 << 20, (1 << 22) + 3])
@pytest.mark.parametrize("spread", [1e-2, 0.0])
def test_large_mean_of_long_rows(spread, d):
    """The sum that the mean comes from has more terms the longer a row is; its error must not.

    The mean is off by c mean|x| at most, c = 43 f for 42 additions of a tree and a multiplication (f = 2^-24), however long the row
    is; so a centred value by e0 = c mean|x| + f |x - mu|, 1 / sd by the relative r = c + rms(e0) / sd + 4 f, and y, whose scale is
    one, by e0 / sd + r |y| + 3 f |y|.
    """
    g = torch.Generator(device=DEV).manual_seed(1)
    x = 1000.1 + spread * torch.randn(3, d, device=DEV, generator=g)
    x64 = x.double()
    c = x64 - x64.mean(-1, keepdim=True)
    sd = (c.square().mean(-1, keepdim=True) + 1e-5).sqrt()
    want = c / sd
    e0 = 43 * F * x64.abs().mean(-1, keepdim=True) + F * c.abs()
    r = 43 * F + e0.square().mean(-1, keepdim=True).sqrt() / sd + 4 * F
    bound = e0 / sd + (r + 3 * F) * want.abs()
    off = (layer_norm(x).double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


# one or two rows per turn of the ring, scalar loads, rows that are read more than once
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [8, 128, 129, 1000, 8192, 8193, 16384, 20000])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
def test_rows_that_are_not_finite(what, d, dtype):
    """Such a row is NaN, and its gradient; no other row changes by a bit.  The sums over rows, which it belongs to, are NaN."""
    g = torch.Generator(device=DEV).manual_seed(2)
    n = 37
    x, dy = (torch.randn(n, d, device=DEV, generator=g).to(dtype) for _ in range(2))
    w = (1 + 0.2 * torch.randn(d, device=DEV, generator=g)).requires_grad_()
    rows = torch.ones(n, dtype=torch.bool, device=DEV)
    rows[[0, 20]] = False

    def run(x, dy):
        x = x.detach().requires_grad_()
        y = layer_norm(x, w)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    want = run(x, dy)
    bad = x.clone()
    bad[0, d // 2] = what
    bad[20, 0] = what
    y, dx, dw = run(bad, dy)
    assert bool(y[~rows].isnan().all()) and bool(dx[~rows].isnan().all()) and bool(dw.isnan().all())
    assert torch.equal(y[rows], want[0][rows]) and torch.equal(dx[rows], want[1][rows])
    worse = dy.clone()
    worse[0, d // 2] = what
    y, dx, dw = run(x, worse)
    assert torch.equal(y, want[0]) and torch.equal(dx[1:], want[1][1:])
    same = torch.arange(d, device=DEV) != d // 2
    assert torch.equal(dw[same], want[2][same]) and not bool(dw[d // 2].isfinite())
