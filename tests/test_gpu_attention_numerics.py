"""Attention where the data's size, not its masks, makes it hard, against the definition in 64 bits."""
import math

import pytest
import torch

from attention_reference import HALF_STEP, reference
from falkon_b200.mmv_ops import attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(b, nq, nk, hq, hk, d, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return tuple(torch.randn(b, n, h, d, device=DEV, generator=g, dtype=dtype) for n, h in ((nq, hq), (nk, hk), (nk, hk), (nq, hq)))


def slopes_of(h):
    return torch.exp2(-8.0 * torch.arange(1, h + 1, device=DEV, dtype=torch.float32) / h)


def worst(got, want, bound):
    """Largest share of its bound that an element is off by."""
    assert got.shape == want.shape and bool(got.isfinite().all())
    return float(((got.double() - want).abs() / bound).max())


def run(q, k, v, do, **opts):
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out, lse = attention(q, k, v, return_lse=True, **opts)
    return dict(zip(("out", "lse", "dq", "dk", "dv"), (out.detach(), lse, *torch.autograd.grad(out, (q, k, v), do))))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cap", [200.0, 1e3, 1e5, 1e6, 1e8, 1e30])
def test_large_caps(cap, d, dtype):
    """A cap far above the scores changes next to nothing, and its size is no measure of what a score may be off.

    Bounds are twice those of the call without a cap.  S = cap tanh(r / cap) costs r seven more roundings (the scaling, at most
    five steps of a polynomial and its fit, the cap), 7 * 2^-24 |S|, where the bound of a score has d 2^-24 |scale| |q||k|^T, which
    is larger; and weights differ from those without a cap by the factor exp(|r|^3 / cap^2), below 1.1 for |r| < 15.
    """
    q, k, v, do = make(1, 260, 260, 4, 2, d, dtype, 1)
    q = q * 2
    for opts in (dict(causal=True), dict(slopes=slopes_of(4)), dict(scale=-0.1, causal=True)):
        want, bounds = reference(q, k, v, do, softcap=cap, **opts), reference(q, k, v, do, **opts)
        got = run(q, k, v, do, softcap=cap, **opts)
        for n in got:
            assert worst(got[n], want[n], bounds["e_" + n]) <= 2, n
    for nq in (1, 3):  # single tokens
        want, bounds = reference(q[:, :nq], k, v, softcap=cap), reference(q[:, :nq], k, v)
        got = dict(zip(("out", "lse"), attention(q[:, :nq], k, v, softcap=cap, return_lse=True)))
        for n in got:
            assert worst(got[n], want[n], bounds["e_" + n]) <= 2, n


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap,size", [(1e4, 2e3), (1e6, 2e5), (300.0, 60.0)])
def test_capped_rows_beside_a_large_one(cap, size, dtype):
    """A row whose scores the cap bends does not cost its neighbours digits (they share a tile, and a warp).  Bounds as above; the
    large row is left to them too, its scores' own bound being large."""
    if dtype == torch.float16 and size > 6e4:
        pytest.skip("beyond fp16")
    q, k, v, do = make(1, 150, 150, 2, 2, 64, dtype, 2)
    q[:, 77] = q[:, 77] / q[:, 77].abs().amax() * size
    want, bounds = reference(q, k, v, do, softcap=cap), reference(q, k, v, do)
    got = run(q, k, v, do, softcap=cap)
    small = torch.arange(150, device=DEV) != 77
    for n in ("out", "dq"):
        assert worst(got[n][:, small], want[n][:, small], bounds["e_" + n][:, small]) <= 2, n
    assert worst(got["lse"][..., small], want["lse"][..., small], bounds["e_lse"][..., small]) <= 2
    token = attention(q[:, 76:79], k, v, softcap=cap)
    assert worst(token[:, ::2], want["out"][:, 76:79:2], bounds["e_out"][:, 76:79:2]) <= 2
