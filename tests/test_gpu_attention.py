"""Attention against its definition in 64 bits, elementwise within the bounds that tests/attention_reference.py derives:
every type, mask and head layout, lengths around the tiles' ends, rows that see nothing, garbage in what is masked."""
import math

import pytest
import torch

from attention_reference import check, reference
from falkon_b200 import _lib
from falkon_b200.mmv_ops import attention, layer_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(b, nq, nk, hq, hk, d, dtype, seed=0, packed=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if packed:
        x = torch.randn(b, nq, hq + 2 * hk, d, device=DEV, generator=g, dtype=dtype)
        q, k, v = x[:, :, :hq], x[:, :, hq:hq + hk], x[:, :, hq + hk:]
    else:
        q = torch.randn(b, nq, hq, d, device=DEV, generator=g, dtype=dtype)
        k = torch.randn(b, nk, hk, d, device=DEV, generator=g, dtype=dtype)
        v = torch.randn(b, nk, hk, d, device=DEV, generator=g, dtype=dtype)
    do = torch.randn(b, nq, hq, d, device=DEV, generator=g, dtype=dtype)
    return q, k, v, do


def run_and_check(q, k, v, do=None, **opts):
    ref = reference(q, k, v, do, **opts)
    if do is None:
        out, lse = attention(q, k, v, return_lse=True, **opts)
        check("out", out, ref)
        check("lse", lse, ref)
        assert torch.equal(out, attention(q, k, v, **opts))
        return out
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out, lse = attention(q, k, v, return_lse=True, **opts)
    grads = torch.autograd.grad(out, (q, k, v), do)
    check("out", out.detach(), ref)
    check("lse", lse, ref)
    for name, t in zip(("dq", "dk", "dv"), grads):
        check(name, t, ref)
    again = torch.autograd.grad(attention(q, k, v, **opts), (q, k, v), do)
    assert all(torch.equal(x, y) for x, y in zip(grads, again)), "another run gave other bits"
    return out


def slopes_of(h):
    return torch.exp2(-8.0 * torch.arange(1, h + 1, device=DEV, dtype=torch.float32) / h)


def docs_of(b, n, lens, pad=0):
    row = torch.cat([torch.full((m,), i) for i, m in enumerate(lens)] + [torch.full((pad,), -1)])
    assert row.numel() == n
    return row.to(torch.int32).to(DEV).expand(b, n).contiguous()


SIZES = [(1, 1, 1, 1, 1, 8), (2, 1, 130, 4, 2, 64), (1, 65, 64, 2, 2, 32), (2, 127, 129, 3, 1, 128), (1, 200, 200, 4, 4, 80),
         (1, 128, 384, 2, 1, 64), (2, 300, 77, 2, 2, 128), (1, 513, 513, 1, 1, 96)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_forward_and_gradients(size, causal, dtype):
    run_and_check(*make(*size, dtype), causal=causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [1, 3, 7, 20, 121])
def test_odd_head_dimensions(d, dtype):
    run_and_check(*make(1, 70, 70, 2, 1, d, dtype), causal=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.0, 2.0, 50.0])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("causal", [False, True])
def test_cap_and_distance_bias(causal, bias, cap, dtype):
    q, k, v, do = make(2, 260, 260, 6, 2, 64, dtype, seed=1)
    run_and_check(q * 3, k, v, do, causal=causal, softcap=cap, slopes=slopes_of(6) if bias else None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [-0.3, 0.0, 0.01, 1.5])
def test_scales(scale, dtype):
    run_and_check(*make(1, 150, 150, 2, 2, 64, dtype, seed=2), scale=scale, softcap=5.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens,pad", [([300], 0), ([1, 127, 172], 0), ([100, 130], 70), ([5] * 60, 0), ([], 300)])
def test_documents(lens, pad, causal, dtype):
    q, k, v, do = make(2, 300, 300, 4, 2, 64, dtype, seed=3)
    docs = docs_of(2, 300, lens, pad)
    for t in (q, k, v, do):  # padding may hold anything
        t[docs < 0] = float("nan")
    out = run_and_check(q, k, v, do, causal=causal, documents=docs, softcap=20.0)
    assert bool((out[docs < 0] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_documents_in_any_order(dtype):
    q, k, v, do = make(2, 333, 333, 2, 1, 128, dtype, seed=4)
    docs = torch.randint(-1, 4, (2, 333), device=DEV, generator=torch.Generator(device=DEV).manual_seed(5))
    run_and_check(q, k, v, do, causal=True, documents=docs)
    q2, k2, v2, do2 = make(2, 40, 333, 2, 1, 128, dtype, seed=6)
    run_and_check(q2, k2, v2, do2, documents=docs, q_documents=docs[:, :40])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("prefix", [[0, 1], [100, 300], [129, -5], [10**6, 128]])
def test_prefix(prefix, dtype):
    q, k, v, do = make(2, 290, 290, 2, 1, 64, dtype, seed=7)
    run_and_check(q, k, v, do, causal=True, prefix_lens=torch.tensor(prefix, device=DEV), slopes=slopes_of(2))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nq", [1, 2, 5, 16, 40, 130])
def test_lengths_with_garbage_behind_them(nq, causal, dtype):
    lens = torch.tensor([0, 1, 63, 64, 200, 257, 300, 10**6, -3], device=DEV)
    b = len(lens)
    q, k, v, do = make(b, nq, 300, 4, 2, 64, dtype, seed=8)
    behind = torch.arange(300, device=DEV)[None, :] >= lens[:, None]
    k[behind] = float("nan")
    v[behind] = float("inf")
    run_and_check(q, k, v, do, causal=causal, kv_lens=lens, slopes=slopes_of(4))
    starts = torch.tensor([0, 5, 100, -70, 17, -500, 299, 1, 2], device=DEV)
    run_and_check(q, k, v, do, causal=causal, kv_lens=lens, q_starts=starts)
    run_and_check(q, k, v, causal=causal, kv_lens=lens, q_starts=starts)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hk,d,nk", [(1, 1, 64, 1), (8, 1, 128, 1000), (16, 2, 128, 4099), (12, 12, 64, 2050), (40, 8, 96, 777),
                                        (20, 1, 80, 515), (3, 3, 8, 9000)])
def test_single_tokens(hq, hk, d, nk, dtype):
    q, k, v, _ = make(3, 1, nk, hq, hk, d, dtype, seed=9)
    lens = torch.tensor([nk, (nk + 1) // 2, 0], device=DEV, dtype=torch.int32)
    run_and_check(q, k, v, kv_lens=lens, softcap=30.0, slopes=slopes_of(hq))
    run_and_check(q, k, v, causal=True)
    docs = (torch.arange(nk, device=DEV) % 3).expand(3, nk)
    run_and_check(q, k, v, causal=True, documents=docs, q_documents=docs[:, :1], kv_lens=lens)


@pytest.mark.parametrize("dtype", TYPES)
def test_single_tokens_equal_the_rows_of_a_prompt(dtype):
    """Prompt, then tokens one by one over the cache: the same rows, within the bounds of both."""
    n, hq, hk, d = 200, 4, 2, 64
    q, k, v, _ = make(2, n, n, hq, hk, d, dtype, seed=10)
    opts = dict(causal=True, softcap=10.0, slopes=slopes_of(hq))
    ref = reference(q, k, v, **opts)
    cache_k, cache_v = torch.full_like(k, math.nan), torch.full_like(v, math.nan)
    rows = []
    for i in range(n):
        cache_k[:, i], cache_v[:, i] = k[:, i], v[:, i]
        rows.append(attention(q[:, i:i + 1], cache_k, cache_v, kv_lens=torch.full((2,), i + 1, device=DEV, dtype=torch.int32), **opts))
    check("out", torch.cat(rows, 1), ref)
    check("out", attention(q, k, v, **opts), ref)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(dtype):
    b, n, hq, hk, d = 2, 140, 4, 2, 64
    q, k, v, do = make(b, n, n, hq, hk, d, dtype, seed=11, packed=True)
    want = run_and_check(q, k, v, do, causal=True)
    # heads before rows, an address that is not aligned, a broadcast batch, a column-major last dimension
    qt, kt, vt = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
    assert torch.equal(want, run_and_check(qt, kt, vt, do, causal=True))
    off = torch.empty(b * n * hq * d + 1, device=DEV, dtype=dtype)[1:].view(b, n, hq, d).copy_(q)
    assert torch.equal(want, run_and_check(off, k, v, do, causal=True))
    cols = k.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(want, run_and_check(q, cols, v, do, causal=True))
    one = k[:1].expand(b, n, hk, d)
    run_and_check(q, one, v[:, :1].expand(b, n, hk, d), do, causal=True)
    # upstream gradients that are broadcast
    qq = q.detach().requires_grad_()
    attention(qq, k, v).sum().backward()
    ref = reference(q, k, v, torch.ones_like(q))
    check("dq", qq.grad, ref)


def test_gradients_against_differences():
    q, k, v, do = make(1, 9, 9, 2, 1, 16, torch.float32, seed=12)
    opts = dict(causal=True, softcap=3.0, slopes=slopes_of(2), prefix_lens=torch.tensor([4], device=DEV))
    qkv = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(attention(*qkv, **opts), qkv, do)
    h = 2.0**-6  # error of a central difference h^2 f''' / 6, of its rounding 2^-22 f / h: both near 1e-4 of the values
    for which, g in enumerate(grads):
        for at in (0, 37, g.numel() - 1):
            ends = []
            for sign in (1, -1):
                moved = [t.detach().clone() for t in (q, k, v)]
                moved[which].view(-1)[at] += sign * h
                ends.append(float((reference(*moved, **opts)["out"] * do.double()).sum()))
            assert abs((ends[0] - ends[1]) / (2 * h) - float(g.reshape(-1)[at])) < 2e-3


def test_only_some_gradients():
    q, k, v, do = make(1, 130, 130, 2, 1, 64, torch.bfloat16, seed=13)
    ref = reference(q, k, v, do)
    for which, name in enumerate(("dq", "dk", "dv")):
        ts = [t.detach().requires_grad_(i == which) for i, t in enumerate((q, k, v))]
        out = attention(*ts)
        check(name, torch.autograd.grad(out, ts[which], do)[0], ref)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,nq,nk", [(0, 5, 5), (2, 0, 5), (2, 5, 0), (1, 0, 0)])
def test_empty(b, nq, nk, dtype):
    q, k, v, do = make(b, nq, nk, 2, 1, 64, dtype)
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    out, lse = attention(q, k, v, causal=True, return_lse=True)
    assert out.shape == q.shape and bool((out == 0).all()) and bool((lse == -math.inf).all())
    grads = torch.autograd.grad(out, (q, k, v), do)
    assert all(g.shape == t.shape and bool((g == 0).all()) for g, t in zip(grads, (q, k, v)))


def test_scores_of_any_size():
    """Scores far from zero, growing along the keys, and masked infinities: the running maximum moves in every tile."""
    for dtype in TYPES:
        n = 700
        q, k, v, do = make(1, n, n, 1, 1, 64, dtype, seed=14)
        k = k * torch.linspace(0.1, 12, n, device=DEV).to(dtype)[None, :, None, None]
        run_and_check(q * 4, k, v, do)
        run_and_check(q * 4, k.flip(1), v, do, causal=True)
        docs = docs_of(1, n, [300, 400])
        k2 = k.clone()
        k2[:, 350:] = 0
        run_and_check(q, k2, v, do, documents=docs)


def test_small_upstream_gradients_in_fp16():
    """Gradients far below one: weights times gradients would leave fp16's range, were they not scaled."""
    q, k, v, do = make(1, 400, 400, 2, 2, 64, torch.float16, seed=15)
    run_and_check(q, k, v, do * 2.0**-10, causal=True)
    run_and_check(q, k, v, do * 2.0**6, causal=True)


def test_other_stream_and_graph():
    q, k, v, do = make(2, 300, 300, 4, 2, 128, torch.bfloat16, seed=16)
    docs = docs_of(2, 300, [100, 200])
    opts = dict(causal=True, documents=docs, softcap=30.0)
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    want = attention(q, k, v, **opts)
    grads = torch.autograd.grad(want, (q, k, v), do)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = attention(q, k, v, **opts)
        g2 = torch.autograd.grad(out, (q, k, v), do)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(want, out) and all(torch.equal(x, y) for x, y in zip(grads, g2))
    want = want.detach()
    del out, g2  # a backward pass is captured only while no eager graph of its leaves lives (torch's rule)
    graphs = []
    for _ in range(2):  # two graphs replayed side by side share nothing
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = attention(q, k, v, **opts)
            g2 = torch.autograd.grad(out, (q, k, v), do)
        graphs.append((graph, out, g2, torch.cuda.Stream()))
    for graph, out, _, st in graphs:
        out.detach().zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, _, _, st in graphs:
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, g2, _ in graphs:
        assert torch.equal(want, out) and all(torch.equal(x, y) for x, y in zip(grads, g2))


def test_normalised_heads_through_attention():
    """A projection's heads, normalised, through attention, forward and backward: the two operators as they are used."""
    b, n, hq, hk, d = 2, 150, 4, 2, 64
    g = torch.Generator(device=DEV).manual_seed(17)
    packed = torch.randn(b, n, hq + 2 * hk, d, device=DEV, generator=g, dtype=torch.float32).requires_grad_()
    w = (1 + 0.2 * torch.randn(2, d, device=DEV, generator=g)).requires_grad_()
    do = torch.randn(b, n, hq, d, device=DEV, generator=g)

    def chain(x, w, norm, attend):
        q, k, v = x[:, :, :hq], x[:, :, hq:hq + hk], x[:, :, hq + hk:]
        return attend(norm(q, w[0]), norm(k, w[1]), v)

    out = chain(packed, w, lambda t, s: layer_norm(t, s), lambda q, k, v: attention(q, k, v, causal=True, softcap=5.0))
    got = torch.autograd.grad(out, (packed, w), do)

    def plain_norm(t, s):
        c = t - t.mean(-1, keepdim=True)
        return c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt() * s

    def plain_attention(q, k, v):
        k, v = (t.repeat_interleave(hq // hk, 2) for t in (k, v))
        s = 5.0 * torch.tanh(torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(d) / 5.0)
        s = s.masked_fill(torch.ones(n, n, device=DEV, dtype=torch.bool).triu(1), -math.inf)
        return torch.einsum("bhij,bjhd->bihd", s.softmax(-1), v)

    x64, w64 = packed.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    ref = chain(x64, w64, plain_norm, plain_attention)
    want = torch.autograd.grad(ref, (x64, w64), do.double())
    # every step is fp32; the longest sums have 2 * 150 * 4 terms: 1200 * 2^-24 = 7e-5 of the largest values
    for a, r in zip((out, *got), (ref, *want)):
        assert float((a.double() - r).abs().max()) <= 1e-4 * float(r.abs().max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,nq,nk,hq,hk,d", [(1, 150, 3001, 2, 1, 128), (1, 40, 5000, 2, 2, 64), (1, 2000, 2000, 2, 1, 64), (2, 1500, 1500, 6, 2, 96)])
def test_long_axes_in_parts(b, nq, nk, hq, hk, d, dtype):
    """Few rows over many keys, few keys under many rows: parts that are worked on apart and joined."""
    q, k, v, do = make(b, nq, nk, hq, hk, d, dtype, seed=18)
    run_and_check(q, k, v, do, causal=True, softcap=20.0)
    if nq == nk:
        lens = [n * nq // 15 for n in (1, 2, 3, 4)]
        docs = docs_of(b, nq, lens + [nq - sum(lens) - 37], 37)
        run_and_check(q, k, v, do, causal=True, documents=docs, slopes=slopes_of(hq))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq", [1, 20, 300])
def test_not_a_number_is_passed_on(nq, dtype):
    """A query that is not a number makes its own row so, and no other; a key that some see, the rows of those that see it."""
    q, k, v, _ = make(1, nq, 300, 2, 1, 64, dtype, seed=19)
    want = attention(q, k, v)
    bad = q.clone()
    bad[0, nq // 2, 1] = float("nan")
    out, lse = attention(bad, k, v, return_lse=True)
    assert bool(out[0, nq // 2, 1].isnan().all()) and bool(lse[0, 1, nq // 2].isnan())
    out[0, nq // 2, 1] = want[0, nq // 2, 1]
    assert torch.equal(out, want)
    worse = k.clone()
    worse[0, 77] = float("nan")
    assert bool(attention(q, worse, v).isnan().all())


def test_offsets_beyond_32_bits():
    """The second sequence lies more than 2^31 elements behind the first."""
    n, hk, d, far = 257, 2, 64, 2**31 + 4096
    room = torch.empty(far + 2 * n * hk * d, device=DEV, dtype=torch.bfloat16)
    k = room.as_strided((2, n, hk, d), (far, hk * d, d, 1))
    v = room.as_strided((2, n, hk, d), (far, hk * d, d, 1), n * hk * d)
    q, k0, v0, do = make(2, n, n, 4, hk, d, torch.bfloat16, seed=20)
    k.copy_(k0)
    v.copy_(v0)
    run_and_check(q, k, v, do, causal=True)
    run_and_check(q[:, :1], k, v, kv_lens=torch.tensor([n, 100], device=DEV))


def test_differentiable_once():
    q, k, v, do = (t.float() for t in make(1, 20, 20, 1, 1, 64, torch.bfloat16, seed=21))
    q.requires_grad_()
    g, = torch.autograd.grad(attention(q, k, v), q, do, create_graph=True)
    with pytest.raises(NotImplementedError, match="once"):
        g.square().sum().backward()
    x = torch.randn(4, 8, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(NotImplementedError, match="once"):
        g.square().sum().backward()


def test_calls_side_by_side():
    """Two streams at once, many times: calls share nothing but the GPU."""
    a = make(2, 300, 300, 4, 2, 64, torch.bfloat16, seed=22)
    b = make(1, 700, 700, 2, 1, 128, torch.bfloat16, seed=23)

    def work(x):
        q, k, v, do = (t.detach().requires_grad_() for t in x)
        out = attention(q, k, v, causal=True)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), do.detach()))

    want = [work(a), work(b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        got = []
        for s, x in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(work(x))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(g, w))


def test_no_wait_gave_up():
    assert _lib.attention_status(torch.device("cuda", torch.cuda.current_device())) == 0


def test_launches_are_counted():
    q, k, v, _ = make(1, 64, 64, 1, 1, 64, torch.bfloat16)
    before = _lib.launch_count()
    attention(q, k, v)
    assert _lib.launch_count() > before


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (3, 3, 128), (6, 2, 32)])
def test_garbage_in_queries_that_see_nothing(hq, hk, d, dtype):
    """Queries before the first key, or of documents without keys, and their output gradients, reach no other row."""
    q, k, v, do = make(2, 200, 230, hq, hk, d, dtype, seed=40)
    starts = torch.tensor([-70, -1000], device=DEV)
    for first, sequence in ((70, 0), (200, 1)):
        q[sequence, :first] = float("nan")
        do[sequence, :first] = float("inf")
    out = run_and_check(q, k, v, do, causal=True, q_starts=starts, softcap=9.0)
    assert not bool(out[0, :70].any()) and not bool(out[1].any())
    q, k, v, do = make(1, 200, 230, hq, hk, d, dtype, seed=41)
    docs, q_docs = (torch.arange(n, device=DEV)[None] // 20 for n in (230, 200))
    q_docs = torch.where(q_docs % 3 == 1, q_docs + 1000, q_docs)
    q[q_docs >= 1000] = float("inf")
    do[q_docs >= 1000] = float("nan")
    run_and_check(q, k, v, do, documents=docs, q_documents=q_docs)
    run_and_check(q, k, v, do, causal=True, q_starts=torch.tensor([30], device=DEV), documents=docs, q_documents=q_docs)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq", [1, 3, 20, 150])
def test_garbage_in_keys_behind_the_last_query(nq, dtype):
    """A causal call over a cache that is longer than what has been written, told by the queries' positions alone."""
    q, k, v, do = make(3, nq, 400, 4, 2, 64, dtype, seed=42)
    starts = torch.tensor([0, 129, 400 - nq], device=DEV)
    prefix = torch.tensor([0, 200, 7], device=DEV)
    for i in range(3):
        reach = max(int(starts[i]) + nq, int(prefix[i]))
        k[i, reach:] = float("nan")
        v[i, reach:] = float("inf")
    run_and_check(q, k, v, do, causal=True, q_starts=starts, prefix_lens=prefix)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("b,n,hq,hk", [(1, 1500, 16, 8), (5, 700, 12, 6), (3, 650, 21, 7), (40, 140, 4, 4)])
def test_documents_of_many_lengths(b, n, hq, hk, causal, dtype):
    """More blocks than SMs: they start in the order of their work, whatever the documents' order in the rows."""
    q, k, v, do = make(b, n, n, hq, hk, 64, dtype, seed=43)
    g = torch.Generator(device="cpu").manual_seed(n)
    lens = [1, 400 % n, 3, 90, 37]
    ids = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
    ids = torch.cat([ids, torch.full((n,), 7)])[:n]
    docs = torch.stack([torch.roll(ids, int(torch.randint(0, n, (1,), generator=g))) for _ in range(b)])
    docs[:, n - 11:n - 4] = -1
    docs = docs.to(DEV)
    run_and_check(q, k, v, do, causal=causal, documents=docs)
    keys = torch.cat([docs, docs[:, :300 % n]], 1)
    k, v = (torch.cat([t, t[:, :300 % n]], 1) for t in (k, v))
    run_and_check(q, k, v, do, causal=causal, documents=keys, q_documents=docs, kv_lens=torch.full((b,), n + 17, device=DEV))


@pytest.mark.parametrize("nq,nk,hq,hk,d", [(100, 3000, 4, 4, 64), (70, 1500, 2, 1, 128), (1, 3000, 16, 1, 64), (2, 2500, 7, 1, 100), (3, 1000, 5, 5, 32),
                                           (16, 700, 2, 2, 128), (17, 700, 2, 2, 64)])
def test_fp32_parts_of_the_key_axis(nq, nk, hq, hk, d):
    q, k, v, do = make(2, nq, nk, hq, hk, d, torch.float32, seed=44)
    lens = torch.tensor([nk - 200, nk], device=DEV)
    docs = (torch.arange(nk, device=DEV) // 300).expand(2, nk)
    run_and_check(q, k, v, do, causal=True, kv_lens=lens, softcap=12.0, slopes=slopes_of(hq))
    run_and_check(q, k, v, do, causal=True, prefix_lens=lens // 2, q_starts=torch.tensor([-1, nk // 3], device=DEV))
    run_and_check(q * 4, k, v, documents=docs, q_documents=docs[:, nk - nq:] - (torch.arange(nq, device=DEV) == 1).long() * 100)
