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


def bits_of(got, part):
    return [part(got["dq"]), part(got["dk"]), part(got["dv"])]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,hq,hk,d", [(100, 2, 2, 64), (400, 6, 2, 128), (1000, 4, 1, 64)])
def test_gradients_owe_nothing_to_other_sequences_and_heads(n, hq, hk, d, dtype):
    """Upstream gradients and values of another sequence, or of another key head's group, may be 10^5 times larger, or infinite:
    the gradients stay what they are, bit by bit."""
    q, k, v, do = make(2, n, n, hq, hk, d, dtype, 3)
    do = do / 16
    want = run(q, k, v, do, causal=True)
    for change in (lambda t: t * 2.0**13, lambda t: t * math.inf):
        d2, v2 = do.clone(), v.clone()
        d2[0] = change(do[0])
        v2[0] = v[0] * 256
        got = run(q, k, v2, d2, causal=True)
        for x, y in zip(bits_of(got, lambda t: t[1]), bits_of(want, lambda t: t[1])):
            assert torch.equal(x, y)
        if hk > 1:
            d2 = do.clone()
            d2[:, :, :hq // hk] = change(do[:, :, :hq // hk])
            got = run(q, k, v, d2, causal=True)
            for n_, first in (("dq", hq // hk), ("dk", 1), ("dv", 1)):
                assert torch.equal(got[n_][:, :, first:], want[n_][:, :, first:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,hq,hk,d", [(200, 2, 2, 64), (500, 4, 2, 128), (900, 4, 1, 64)])
def test_gradients_owe_nothing_to_other_rows(n, hq, hk, d, dtype):
    """The same within a sequence: queries of its first part, and documents beside one another in a tile."""
    q, k, v, do = make(1, n, n, hq, hk, d, dtype, 4)
    do = do / 16
    cut = n // 2 + 5
    large = do.clone()
    large[:, :cut] *= 2.0**13
    want, got = run(q, k, v, do, causal=True), run(q, k, v, large, causal=True)
    for x, y in zip(bits_of(got, lambda t: t[:, cut:]), bits_of(want, lambda t: t[:, cut:])):  # keys that only later queries see
        assert torch.equal(x, y)
    docs = torch.arange(n, device=DEV)[None] // 37
    even = (docs[0] % 2 == 0)
    large = torch.where(even[None, :, None, None], do * 2.0**13, do)
    big_v = torch.where(even[None, :, None, None], v * 256, v)
    want, got = run(q, k, v, do, documents=docs), run(q, k, big_v, large, documents=docs)
    for x, y in zip(bits_of(got, lambda t: t[:, ~even]), bits_of(want, lambda t: t[:, ~even])):
        assert torch.equal(x, y)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("growth", [2.0**0.03, 2.0**-0.03])
def test_fp16_gradients_that_grow_along_a_row(growth, d):
    """Terms of dK and dV grow, or shrink, by 2^18 from the first query tile to the last, and those of dQ along the keys: the
    factor that a row is held with follows.  A row keeps the bounds that it has when the smaller terms are not there to be lost:
    2^-29 of the largest term for each of 600 terms is far below the rounding of the largest one, 2^-11."""
    n = 600
    q, k, v, do = make(1, n, n, 2, 1, d, torch.float16, 5)
    f = growth ** torch.arange(n, device=DEV, dtype=torch.float64)
    f = (f / f.max() * 2.0**6).to(torch.float32)[None, :, None, None]
    for do2, v2 in ((do * f, v), (do, v * f), (do * f, v * f)):
        do2, v2 = do2.half(), v2.half()
        want, got = reference(q, k, v2, do2, causal=growth < 1), run(q, k, v2, do2, causal=growth < 1)
        for name in ("out", "dq", "dk", "dv"):
            assert worst(got[name], want[name], want["e_" + name]) <= 1, name


@pytest.mark.parametrize("dtype", TYPES)
def test_labels_beyond_int32(dtype):
    """They mark padding: two documents never become one, and the largest label that is one stays apart from them."""
    q, k, v, do = make(1, 200, 200, 2, 1, 64, dtype, 6)
    docs = torch.tensor([3, 2**31 - 1, 2**31, 2**40], device=DEV).repeat_interleave(50)[None]
    out = run(q, k, v, do, documents=docs)
    same = run(q, k, v, do, documents=torch.tensor([0, 1, -1, -1], device=DEV, dtype=torch.int32).repeat_interleave(50)[None])
    for n in out:
        assert torch.equal(out[n], same[n]), n
    assert not bool(out["out"][:, 100:].any()) and bool((out["lse"][..., 100:] == -math.inf).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,nq,nk,hq,hk", [(1, 8192, 1 << 18, 16, 1), (222, 1, 1 << 16, 8, 8)])
def test_many_small_weights_beside_a_large_one(b, nq, nk, hq, hk, dtype):
    """One key has most of the weight, and each of very many others a 2^-25th of it, half of fp16's smallest step: held as they are
    they would be lost, though together they make 2^-7 (or 2^-9) of the sum.  The key axis is in one part here.  The large key's
    value is zero, so the result is the small ones' share.  Relative error: u for the result, 2^-7 for the weights (which have at
    least 6 bits), and nk steps of fp32 for a sum of nk equal terms in any order, each addition cut or rounded.
    """
    gap = torch.tensor(17.35).to(dtype)
    q, k, v = (torch.zeros(b, n, h, 8, device=DEV, dtype=dtype) for n, h in ((nq, hq), (nk, hk), (nk, hk)))
    q[..., 0] = 1
    k[:, 5, :, 0] = gap
    v[:] = 1
    v[:, 5] = 0
    small = (nk - 1) * math.exp(-float(gap))
    assert 2.0**-10 < small < 2.0**-6
    want, lse = small / (small + 1), float(gap) + math.log1p(small)
    out, got = attention(q, k, v, scale=1.0, return_lse=True)
    assert float((out.double() - want).abs().max()) <= want * (HALF_STEP[dtype] + 2.0**-7 + nk * 2.0**-23)
    assert float((got.double() - lse).abs().max()) <= 2.0**-18 + nk / 16 * 2.0**-24


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nq,nk", [(1, 300), (20, 300), (300, 200)])
def test_positions_far_from_all_keys(nq, nk, causal, dtype):
    """A distance that every pair of a sequence has changes no weight and no gradient: queries far behind all keys, or before them,
    get what queries next to the keys get, within those queries' bounds.  The log-sum-exp has the distance in it, and fp32's step
    of that."""
    q, k, v, do = make(5, nq, nk, 4, 2, 64, dtype, 7)
    lens = torch.tensor([nk, nk, nk - 77, nk, nk - 20], device=DEV)
    far = torch.tensor([10**6, 2**29, 300000, nk - nq, 2**40], device=DEV)
    near = torch.tensor([nk - 1, nk - 1, nk - 78, nk - nq, nk - 21], device=DEV)
    if not causal:
        far[3], near[3] = -(10**7), -nq
    slopes = slopes_of(4)
    opts = dict(causal=causal, kv_lens=lens, slopes=slopes)
    want = reference(q, k, v, do, q_starts=near, **opts)
    got = run(q, k, v, do, q_starts=far, **opts)
    for n in ("out", "dq", "dk", "dv"):
        assert worst(got[n], want[n], want["e_" + n]) <= 1, n
    shift = slopes.double()[:, None] * (far.clamp(-(2**29), 2**29) - near).abs()[:, None, None]
    some = want["lse"].isfinite()  # of queries that see a key
    assert torch.equal(got["lse"].isfinite(), some)
    assert worst(got["lse"][some], (want["lse"] - shift)[some], (want["e_lse"] + 2.0**-23 * (want["lse"].abs() + shift))[some]) <= 1
    assert torch.equal(got["out"], attention(q, k, v, q_starts=far, **opts))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nq,nk,hq,hk,d", [(300, 300, 4, 2, 128), (300, 300, 3, 3, 64), (40, 900, 2, 1, 64), (16, 5000, 4, 1, 128), (1, 700, 8, 2, 80)])
def test_what_rounding_takes_from_the_output_is_kept(nq, nk, hq, hk, d, dtype):
    """Equal scores make the weights exact, and the output a mean of values in fp32: it and what rounding took from it, which the
    backward pass adds back, together miss it by the rounding of what was taken, u (u |out|), and of nk additions."""
    q, k, v, do = make(2, nq, nk, hq, hk, d, dtype, 8)
    q = torch.zeros_like(q).requires_grad_()
    u = HALF_STEP[dtype]
    for opts in (dict(), dict(causal=True), dict(documents=(torch.arange(nk, device=DEV) // 50).expand(2, nk),
                                                 q_documents=(torch.arange(nq, device=DEV) // 50).expand(2, nq))):
        out = attention(q, k, v, **opts)
        hi, lo = out.grad_fn.saved_tensors[3:5]
        hi, lo = hi[..., :d].double(), lo[..., :d].double()
        want, size = reference(q, k, v, **opts)["out"], reference(q, k, v.abs(), **opts)["out"]
        assert torch.equal(hi, out.detach().double()) and bool((lo.abs() <= u * hi.abs() + 2.0**-25).all())
        tiny = 2.0**-25 if dtype == torch.float16 else 0.0  # half of the smallest step, for the remainder too
        assert bool(((hi + lo - want).abs() <= u * u * want.abs() * 1.01 + nk * 2.0**-23 * size + tiny + 1e-30).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,hq,hk,d", [(2, 2, 2, 64), (8, 4, 2, 128), (64, 3, 1, 64), (256, 2, 1, 128)])
def test_gradients_of_few_keys_that_cancel(n, hq, hk, d, dtype):
    """Equal scores of 2^m keys: weights are exact, so what dq and dk miss comes from dS alone.  Its row adds up to zero, and a vector
    that all keys share, 32 times as large as what tells them apart, leaves nothing but errors of dS, and of dout . out; so do
    queries that come in pairs of opposite sign with the same upstream gradient.  dS and its remainder miss u u |dS| (twice: the
    remainder is rounded, and what the product's fp32 sums cut is no more), and the fp32 sums of dP and delta d 2^-24 of their terms.
    """
    u = HALF_STEP[dtype]
    _, k, v, do = make(2, n, n, hq, hk, d, dtype, 9)
    shift = torch.randn(2, 1, hk, d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(10)).to(dtype) * 32
    zero = torch.zeros(2, n, hq, d, device=DEV, dtype=dtype)
    sign = (1 - 2 * (torch.arange(n, device=DEV) % 2)).to(dtype)[None, :, None, None]
    pairs = torch.randn(2, 1, hq, d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(11)).to(dtype) * 32 * sign
    same = do[:, ::2].repeat_interleave(2, 1)
    for which, q2, k2, do2 in (("dq", zero, k + shift, do), ("dk", pairs, torch.zeros_like(k), same)):
        want, got = reference(q2, k2, v, do2), run(q2, k2, v, do2)
        D, V = do2.double(), v.double().repeat_interleave(hq // hk, 2)
        P = 1.0 / n
        dP = torch.einsum("bihd,bjhd->bhij", D, V)
        dS = (P * (dP - dP.mean(-1, keepdim=True))).abs()
        size = torch.einsum("bihd,bjhd->bhij", D.abs(), V.abs())
        e = (2 * u * u + 2.0**-19) * dS + P * d * 2.0**-23 * (size + size.mean(-1, keepdim=True)) + (n + 4) * 2.0**-23 * dS
        if dtype == torch.float16:
            e = e + 2.0**-28 * dS.amax((-1, -2), keepdim=True)  # the lower end of fp16 under a row's factor
        scale = 1 / math.sqrt(d)
        if which == "dq":
            bound = scale * torch.einsum("bhij,bjhd->bihd", e, k2.double().abs().repeat_interleave(hq // hk, 2))
        else:
            bound = scale * torch.einsum("bhij,bihd->bjhd", e, q2.double().abs()).unflatten(2, (hk, hq // hk)).sum(3)
        bound = bound + u * want[which].abs() + (2.0**-25 if dtype == torch.float16 else 0.0) + 1e-30
        assert worst(got[which], want[which], bound) <= 1, which


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq,hq", [(1, 2), (3, 4), (30, 2)])
def test_distances_behind_the_16_millionth_key(nq, hq, dtype):
    """fp32 has no odd numbers beyond 2^24: distances are taken between whole numbers.  With a slope of one only the last keys have
    weight (what lies 300 keys back has less than e^-200 of it), so the call on those alone is the reference."""
    nk, last = 2**24 + 1001, 400
    g = torch.Generator(device=DEV).manual_seed(12)
    k, v = (torch.zeros(1, nk, 1, 8, device=DEV, dtype=dtype) for _ in range(2))
    for t in (k, v):
        t[:, -last:] = torch.randn(1, last, 1, 8, device=DEV, generator=g, dtype=dtype)
    q = torch.randn(1, nq, hq, 8, device=DEV, generator=g, dtype=dtype)
    slopes = torch.ones(hq, device=DEV)
    out = attention(q, k, v, causal=True, slopes=slopes)
    want = reference(q, k[:, -last:], v[:, -last:], causal=True, slopes=slopes)
    assert worst(out, want["out"], want["e_out"]) <= 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,nq,nk", [(0, 5, 5), (2, 0, 5), (2, 5, 0), (1, 0, 0)])
def test_documents_of_nothing(b, nq, nk, dtype):
    q, k, v, do = make(b, nq, nk, 2, 1, 64, dtype, 13)
    docs, q_docs = (torch.zeros(b, n, device=DEV, dtype=torch.int32) for n in (nk, nq))
    got = run(q, k, v, do, causal=True, documents=docs, q_documents=q_docs)
    assert got["out"].shape == q.shape and bool((got["lse"] == -math.inf).all())
    assert not any(bool(got[n].any()) for n in ("out", "dq", "dk", "dv"))
