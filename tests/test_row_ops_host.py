"""Refusals of ``attention`` and ``layer_norm`` and of their C entry points, before anything reaches a GPU."""
import ctypes
import sys

import pytest
import torch

from falkon_b200 import _lib, mmv_ops
from falkon_b200.mmv_ops import attention, layer_norm


@pytest.fixture(scope="module")
def lib():
    _lib.build()
    return _lib.load()


@pytest.fixture
def gpu_claimed(monkeypatch):
    """The checks in front of the first CUDA call run on a machine without a GPU too."""
    for name in ("attention", "layer_norm"):  # the package's attributes of these names are the functions
        monkeypatch.setattr(sys.modules["falkon_b200.mmv_ops." + name], "_require_cuda", lambda *a: None)


def qkv(b=1, nq=4, nk=4, hq=2, hk=1, d=16, dtype=torch.float32):
    return torch.zeros(b, nq, hq, d, dtype=dtype), torch.zeros(b, nk, hk, d, dtype=dtype), torch.zeros(b, nk, hk, d, dtype=dtype)


def test_exported():
    assert "attention" in mmv_ops.__all__ and "layer_norm" in mmv_ops.__all__


@pytest.mark.parametrize("change,error", [
    (lambda q, k, v: (q[0], k, v), ValueError), (lambda q, k, v: (q.numpy(), k, v), TypeError), (lambda q, k, v: (q.double(), k, v), TypeError),
    (lambda q, k, v: (q.double(), k.double(), v.double()), TypeError), (lambda q, k, v: (q, k.half(), v), TypeError),
    (lambda q, k, v: (q, k[:, :3], v), ValueError), (lambda q, k, v: (q[..., :8], k, v), ValueError),
    (lambda q, k, v: (q.repeat(1, 1, 1, 9), k.repeat(1, 1, 1, 9), v.repeat(1, 1, 1, 9)), NotImplementedError),
    (lambda q, k, v: (torch.zeros(1, 4, 3, 16), k.repeat(1, 1, 2, 1), v.repeat(1, 1, 2, 1)), ValueError),
    (lambda q, k, v: (q, k, v), ValueError),  # host tensors
])
def test_attention_operands(change, error, gpu_claimed):
    with pytest.raises(error):
        attention(*change(*qkv()))


@pytest.mark.parametrize("opts,error", [
    (dict(scale=float("nan")), ValueError), (dict(scale=float("inf")), ValueError), (dict(softcap=-1.0), ValueError), (dict(softcap=float("nan")), ValueError),
    (dict(slopes=torch.zeros(3)), ValueError), (dict(slopes=torch.zeros(2, dtype=torch.float64)), ValueError),
    (dict(slopes=torch.zeros(2, requires_grad=True)), NotImplementedError),
    (dict(prefix_lens=torch.zeros(1, dtype=torch.int32)), ValueError),
    (dict(q_documents=torch.zeros(1, 4, dtype=torch.int32)), ValueError),
    (dict(documents=torch.zeros(1, 5, dtype=torch.int32)), ValueError), (dict(documents=torch.zeros(1, 4)), TypeError),
    (dict(kv_lens=torch.zeros(2, dtype=torch.int32)), ValueError), (dict(kv_lens=torch.zeros(1)), TypeError), (dict(kv_lens=[4]), TypeError),
    (dict(q_starts=torch.zeros(1, dtype=torch.int16)), TypeError),
])
def test_attention_options(opts, error, gpu_claimed, monkeypatch):
    class Cuda(torch.Tensor):  # tensors that say they are on a GPU get past the device check; nothing may be launched
        device = torch.device("cuda", 0)

    def on_gpu(t):
        return t.as_subclass(Cuda) if isinstance(t, torch.Tensor) else t

    monkeypatch.setattr(_lib, "call_rows", lambda *a: pytest.fail("a refused call reached the library"))
    with pytest.raises(error):
        attention(*map(on_gpu, qkv()), **{n: on_gpu(t) for n, t in opts.items()})


def test_documents_need_the_queries_own(gpu_claimed, monkeypatch):
    class Cuda(torch.Tensor):
        device = torch.device("cuda", 0)

    ts = [t.as_subclass(Cuda) for t in qkv(nq=2)]
    with pytest.raises(ValueError, match="q_documents"):
        attention(*ts, documents=torch.zeros(1, 4, dtype=torch.int32).as_subclass(Cuda))


@pytest.mark.skipif(torch.cuda.is_available(), reason="needs a machine without a GPU")
def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="CUDA device"):
        attention(*qkv())
    with pytest.raises(RuntimeError, match="CUDA device"):
        layer_norm(torch.zeros(3, 4))


@pytest.mark.parametrize("args,error", [
    ((torch.zeros(3, 4),), ValueError), ((torch.zeros(3, 4).double(),), TypeError), ((torch.zeros(3, 0),), ValueError), ((torch.tensor(1.0),), ValueError),
    (([1.0],), TypeError), ((torch.zeros(3, 4), None, None, -1.0), ValueError), ((torch.zeros(3, 4), None, None, float("nan")), ValueError),
])
def test_layer_norm_operands(args, error, gpu_claimed):
    with pytest.raises(error):
        layer_norm(*args)


@pytest.mark.parametrize("w,b,error", [
    (torch.zeros(5), None, ValueError), (torch.zeros(4, dtype=torch.float64), None, TypeError), (None, torch.zeros(4, 1), ValueError),
    (torch.zeros(4), torch.zeros(4, dtype=torch.bfloat16), TypeError), ([1.0] * 4, None, TypeError),
])
def test_layer_norm_weights(w, b, error, gpu_claimed):
    class Cuda(torch.Tensor):
        device = torch.device("cuda", 0)

    ts = [t.as_subclass(Cuda) if isinstance(t, torch.Tensor) else t for t in (torch.zeros(3, 4, dtype=torch.bfloat16), w, b)]
    with pytest.raises(error):
        layer_norm(*ts)


# ---------------------------------------------------------------------------------------------------------------------
# C entry points: status codes before anything is launched
# ---------------------------------------------------------------------------------------------------------------------
def attention_args(**change):
    t = _lib.Tensor4(4096, 4 * 2 * 64, 2 * 64, 64)
    kv = _lib.Tensor4(4096, 4 * 64, 64, 64)
    a = _lib.AttentionArgs(_lib.FLK_BF16, 1, 4, 4, 2, 1, 64, 0, 0, 0.125, 0.0, t, kv, kv, t)
    a.lse = 4096
    a.dout, a.dq, a.dk, a.dv = t, t, kv, kv
    for n, x in change.items():
        setattr(a, n, x)
    return ctypes.byref(a)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=_lib.FLK_F64), _lib.FLK_ERR_BAD_ARG), (dict(dtype=9), _lib.FLK_ERR_BAD_ARG), (dict(nq=-1), _lib.FLK_ERR_BAD_ARG),
    (dict(flags=1), _lib.FLK_ERR_BAD_ARG), (dict(nq=2**28, hq=8, hk=8), _lib.FLK_ERR_UNSUPPORTED), (dict(hk=0), _lib.FLK_ERR_BAD_ARG), (dict(hq=3, hk=2), _lib.FLK_ERR_BAD_ARG), (dict(d=0), _lib.FLK_ERR_BAD_ARG),
    (dict(d=136), _lib.FLK_ERR_UNSUPPORTED), (dict(d=12), _lib.FLK_ERR_UNSUPPORTED), (dict(nk=2**30), _lib.FLK_ERR_UNSUPPORTED),
    (dict(batch=70000), _lib.FLK_ERR_UNSUPPORTED), (dict(scale=float("nan")), _lib.FLK_ERR_BAD_ARG), (dict(softcap=-1.0), _lib.FLK_ERR_BAD_ARG),
    (dict(q_documents=4096), _lib.FLK_ERR_BAD_ARG), (dict(prefix_lens=4096), _lib.FLK_ERR_BAD_ARG),
    (dict(q=_lib.Tensor4(None, 0, 0, 0)), _lib.FLK_ERR_BAD_ARG), (dict(k=_lib.Tensor4(4098, 0, 64, 64)), _lib.FLK_ERR_LAYOUT),
    (dict(v=_lib.Tensor4(4096, 0, 65, 64)), _lib.FLK_ERR_LAYOUT), (dict(out=_lib.Tensor4(4096, 0, 128, 60)), _lib.FLK_ERR_LAYOUT),
    (dict(q_documents=4096, k_documents=4096), _lib.FLK_ERR_WORKSPACE),
    (dict(q_documents=4096, k_documents=4096, workspace=4100, workspace_bytes=1 << 30), _lib.FLK_ERR_WORKSPACE),
    (dict(q_documents=4096, k_documents=4096, workspace=4096, workspace_bytes=64), _lib.FLK_ERR_WORKSPACE),
])
def test_attention_status(lib, change, status):
    assert lib.flk_attention_forward(attention_args(**change), None) == status
    assert lib.flk_last_error()
    assert lib.flk_attention_backward(attention_args(**change), None) == status
    if status in (_lib.FLK_ERR_BAD_ARG, _lib.FLK_ERR_UNSUPPORTED) and "q" not in change:
        assert lib.flk_attention_workspace_bytes(attention_args(**change), 1) == status


def test_attention_backward_status(lib):
    none = _lib.Tensor4(None, 0, 0, 0)
    for change in (dict(dk=none), dict(dv=none), dict(dout=none), dict(lse=None)):
        assert lib.flk_attention_backward(attention_args(**change), None) == _lib.FLK_ERR_BAD_ARG, change
    assert lib.flk_attention_backward(attention_args(), None) == _lib.FLK_ERR_WORKSPACE
    assert lib.flk_attention_forward(None, None) == _lib.FLK_ERR_BAD_ARG
    assert lib.flk_attention_workspace_bytes(None, 0) == _lib.FLK_ERR_BAD_ARG


def test_nothing_to_do(lib):
    assert lib.flk_attention_forward(attention_args(batch=0), None) == 0
    assert lib.flk_attention_forward(attention_args(nq=0), None) == 0
    assert lib.flk_attention_backward(attention_args(batch=0), None) == 0


def norm_args(**change):
    a = _lib.LayerNormArgs(_lib.FLK_BF16, _lib.FLK_F32, 8, 64, 1e-5, 4096, 1, 64, 0, 4096, 4096, 4096, None, None)
    a.mean = a.rstd = a.dy = a.dx = a.dweight = a.dbias = 4096
    a.dy_inner, a.dy_outer_stride = 1, 64
    for n, x in change.items():
        setattr(a, n, x)
    return ctypes.byref(a)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=_lib.FLK_F64), _lib.FLK_ERR_BAD_ARG), (dict(wdtype=_lib.FLK_F16), _lib.FLK_ERR_BAD_ARG), (dict(n=-1), _lib.FLK_ERR_BAD_ARG),
    (dict(d=0), _lib.FLK_ERR_BAD_ARG), (dict(d=1 << 25), _lib.FLK_ERR_BAD_ARG), (dict(eps=-1.0), _lib.FLK_ERR_BAD_ARG),
    (dict(x_inner=0), _lib.FLK_ERR_BAD_ARG), (dict(x=None), _lib.FLK_ERR_BAD_ARG),
])
def test_layer_norm_status(lib, change, status):
    assert lib.flk_layer_norm_forward(norm_args(**change), None) == status
    assert lib.flk_layer_norm_backward(norm_args(**change), None) == status


def test_layer_norm_workspace(lib):
    assert lib.flk_layer_norm_workspace_bytes(norm_args(dweight=None, dbias=None)) == 0
    need = lib.flk_layer_norm_workspace_bytes(norm_args())
    assert need >= 2 * 64 * 4
    for ws, size in ((None, 0), (4096, need - 1), (4100, need)):
        assert lib.flk_layer_norm_backward(norm_args(workspace=ws, workspace_bytes=size), None) == _lib.FLK_ERR_WORKSPACE
    assert lib.flk_layer_norm_forward(norm_args(n=0), None) == 0
    assert lib.flk_layer_norm_forward(norm_args(mean=None), None) == _lib.FLK_ERR_BAD_ARG
    assert lib.flk_layer_norm_forward(None, None) == _lib.FLK_ERR_BAD_ARG


@pytest.mark.parametrize("scale,softcap", [(0.125, 1e-38), (0.125, 1e-40), (1e10, 1e-25), (-1e10, 1e-25)])
def test_softcap_that_fp32_cannot_hold(lib, scale, softcap):
    change = dict(scale=scale, softcap=softcap)
    assert lib.flk_attention_forward(attention_args(**change), None) == _lib.FLK_ERR_UNSUPPORTED
    assert lib.flk_attention_backward(attention_args(**change), None) == _lib.FLK_ERR_UNSUPPORTED
    assert lib.flk_attention_workspace_bytes(attention_args(**change), 0) == _lib.FLK_ERR_UNSUPPORTED


def test_rows_up_to_a_tile_behind_the_last(lib):
    for change in (dict(nq=2**29 - 1, hq=4, hk=4), dict(nk=2**29 - 1, hq=4, hk=4)):
        assert lib.flk_attention_workspace_bytes(attention_args(**change), 0) == _lib.FLK_ERR_UNSUPPORTED
    assert lib.flk_attention_workspace_bytes(attention_args(nq=2**29 - 256, hq=4, hk=4), 0) >= 0
