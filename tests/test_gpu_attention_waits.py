"""Waits inside the tensor-core attention kernels that run out, because their limit is short or what they wait for never comes."""
import concurrent.futures

import pytest
import torch

from falkon_b200 import _lib
from falkon_b200.mmv_ops import attention

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture
def wait_limit():
    yield _lib.attention_wait_limit
    _lib.attention_wait_limit(1000000000)


def call(shape, dtype, **opts):
    b, nq, nk, hq, hk, d = shape
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, v, do = (torch.randn(b, n, h, d, device=DEV, generator=g, dtype=dtype) for n, h in ((nq, hq), (nk, hk), (nk, hk), (nq, hq)))
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    return q, k, v, do, lambda: attention(q, k, v, return_lse=True, **opts)


# two row tiles a block, one row tile, parts of the key axis, heads of 64 and of 128
SHAPES = [(2, 300, 300, 4, 2, 128), (1, 60, 700, 2, 2, 64), (1, 40, 5000, 2, 1, 128), (3, 1000, 1000, 4, 4, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_no_time_at_all(shape, dtype, wait_limit):
    """No product is issued, so every block with work gives up: all is NaN, the status says so once, and the next call is right."""
    device = torch.device("cuda", torch.cuda.current_device())
    q, k, v, do, forward = call(shape, dtype, causal=True, softcap=20.0)
    want, lse = forward()
    grads = torch.autograd.grad(want, (q, k, v), do, retain_graph=True)
    assert _lib.attention_status(device) == 0
    wait_limit(0)
    out, bad_lse = forward()
    bad_grads = torch.autograd.grad(want, (q, k, v), do, retain_graph=True)  # of the right output
    torch.cuda.synchronize()
    wait_limit(1000000000)
    assert bool(out.isnan().all()) and bool(bad_lse.isnan().all())
    for g, w in zip(bad_grads, grads):  # a key that no query tile meets has no wait in front of its zeros
        assert bool((g.isnan() | (w == 0)).all())
    assert _lib.attention_status(device) == 1 and _lib.attention_status(device) == 0
    again, again_lse = forward()
    assert torch.equal(again, want) and torch.equal(again_lse, lse)
    assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(again, (q, k, v), do), grads))
    assert _lib.attention_status(device) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_some_time(shape, dtype, wait_limit):
    """Limits that run out anywhere in a block's life, or not at all: an element is right or NaN, and NaN only where the status
    tells."""
    device = torch.device("cuda", torch.cuda.current_device())
    q, k, v, do, forward = call(shape, dtype, causal=True, slopes=torch.full((shape[3],), 0.1, device=DEV))
    want, lse = forward()
    grads = torch.autograd.grad(want, (q, k, v), do, retain_graph=True)
    _lib.attention_status(device)
    for ns in (300, 700, 1000, 1500, 2000, 3000, 5000, 20000):
        wait_limit(ns)
        out, got_lse = forward()
        got = torch.autograd.grad(want, (q, k, v), do, retain_graph=True)
        torch.cuda.synchronize()
        wait_limit(1000000000)
        gave_up, lost = _lib.attention_status(device), False
        for x, y in zip((out, got_lse, *got), (want, lse, *grads)):
            lost = lost or bool(x.isnan().any())
            assert bool((x.isnan() | (x == y)).all()), ns
        assert gave_up or not lost


def test_status_queries_side_by_side(wait_limit):
    """What gave up is told to one of the queries that are made at the same time."""
    device = torch.device("cuda", torch.cuda.current_device())
    *_, forward = call((1, 300, 300, 2, 2, 64), torch.bfloat16)
    forward()
    _lib.attention_status(device)
    for _ in range(20):
        wait_limit(0)
        forward()
        torch.cuda.synchronize()
        wait_limit(1000000000)

        def query(_):
            with torch.cuda.stream(torch.cuda.Stream(device)):
                return _lib.attention_status(device)

        with concurrent.futures.ThreadPoolExecutor(4) as pool:
            assert sum(pool.map(query, range(4))) == 1
