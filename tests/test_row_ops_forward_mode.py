"""Forward-mode differentiation and ``torch.func`` transforms of ``attention`` and ``layer_norm``: refused, never dropped."""
import pytest
import torch
from torch.autograd import forward_ad

from falkon_b200.mmv_ops import attention, layer_norm
from falkon_b200.mmv_ops.utils import refuse_tangents

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]  # on the host they are refused before the host is


def qkv(device):
    g = torch.Generator().manual_seed(1)
    return tuple(torch.randn(1, 5, 2, 16, generator=g).to(device) for _ in range(3))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_attention_of_dual_tensors(which, device):
    ts = [*qkv(device), torch.ones(2, device=device)]
    with forward_ad.dual_level():
        ts[which] = forward_ad.make_dual(ts[which], torch.ones_like(ts[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            attention(*ts[:3], slopes=ts[3])
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            attention(*ts[:3], slopes=ts[3])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", [0, 1, 2])
def test_layer_norm_of_dual_tensors(which, device):
    ts = [torch.randn(3, 8, device=device), torch.ones(8, device=device), torch.zeros(8, device=device)]
    with forward_ad.dual_level():
        ts[which] = forward_ad.make_dual(ts[which], torch.ones_like(ts[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            layer_norm(*ts)


def test_tensors_without_a_tangent_pass():
    x = torch.ones(3)
    refuse_tangents("f", x, None, 3.0)
    with forward_ad.dual_level():
        refuse_tangents("f", x, None, 3.0)
        with pytest.raises(NotImplementedError, match="f has no"):
            refuse_tangents("f", None, forward_ad.make_dual(x, x))


@pytest.mark.gpu
def test_tangents_of_upstream_gradients():
    q, k, v = (t.requires_grad_() for t in qkv("cuda"))
    x = torch.randn(3, 8, device="cuda", requires_grad=True)
    for leaves, out in (((q, k, v), attention(q, k, v)), ((x,), layer_norm(x))):
        with forward_ad.dual_level():
            up = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(out, leaves, up)


@pytest.mark.gpu
def test_calls_inside_a_dual_level():
    q, k, v = qkv("cuda")
    x = torch.randn(3, 8, device="cuda")
    want = attention(q, k, v), layer_norm(x)
    with forward_ad.dual_level():
        assert torch.equal(attention(q, k, v), want[0]) and torch.equal(layer_norm(x), want[1])
        q.requires_grad_()
        assert torch.equal(attention(q, k, v), want[0])


@pytest.mark.gpu
def test_function_transforms():
    q, k, v = qkv("cuda")
    x = torch.randn(3, 8, device="cuda")
    for f, t in ((lambda t: attention(t, k, v), q), (lambda t: layer_norm(t), x)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.grad(lambda u: f(u).sum())(t)
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(f, (t,), (torch.ones_like(t),))
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.vmap(f)(t[None])
