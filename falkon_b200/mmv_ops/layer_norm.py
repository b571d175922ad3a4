"""``layer_norm``: rows brought to mean zero and variance one, with a learned scale and shift, and their gradients.

Products compare rows (``fmmv`` by distances in units of sigma, ``attention`` by dot products); this prepares them.  One
kernel of ``libfalkon_b200`` each way (include/falkon_b200.h), and one that adds up the gradients of scale and shift.  There
is no CPU path.
"""
from typing import Optional

import torch

from .. import _lib
from .fmmv import _require_cuda
from .utils import differentiable_once, refuse_tangents

__all__ = ("layer_norm", "LayerNormFn")


def _rows(t: torch.Tensor):
    """``t`` as rows with a two-level index: (tensor, rows, inner, outer stride, inner stride), with a copy only where the
    strides of ``t`` have no such form."""
    d = t.shape[-1]
    n = t.numel() // d
    if t.is_contiguous():
        return t, n, 1, d, 0
    if t.stride(-1) == 1 or d == 1:
        levels = []  # (size, stride) of the leading dimensions, merged from the innermost outwards
        for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if size == 1:
                continue
            if levels and stride == levels[-1][0] * levels[-1][1]:
                levels[-1] = (levels[-1][0] * size, levels[-1][1])
            else:
                levels.append((size, stride))
        if len(levels) < 2:
            return t, n, 1, (levels[0][1] if levels else d), 0
        if len(levels) == 2:
            return t, n, levels[0][0], levels[1][1], levels[0][1]
    return t.contiguous(), n, 1, d, 0


def _ptr(t: Optional[torch.Tensor]):
    return 0 if t is None else t.data_ptr()


def _dense_like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _forward(x, weight, bias, eps, with_stats):
    x, n, inner, so, si = _rows(x)
    y = _dense_like(x)
    stats = torch.empty((2, n), dtype=torch.float32, device=x.device) if with_stats else None
    if n > 0:
        mean = 0 if stats is None else stats.data_ptr()
        code = _lib.row_dtype_code(x.dtype)
        w = weight if weight is not None else bias
        head = _lib._LAYER_NORM_HEAD.pack(
            code, code if w is None else _lib.row_dtype_code(w.dtype), n, x.shape[-1], eps, x.data_ptr(), inner, so, si,
            _ptr(weight), _ptr(bias), y.data_ptr(), mean, mean and mean + 4 * n, 0, 1, 0, 0, 0, 0, 0)
        _lib.call_rows(_lib.load().flk_layer_norm_forward, head, x.device)
    return y, stats


def _backward(ctx, dy):
    refuse_tangents("layer_norm", dy)
    x, weight, stats = ctx.saved_tensors
    need_x, need_w, need_b, _ = ctx.needs_input_grad
    d, dev = x.shape[-1], x.device
    dx = _dense_like(x) if need_x else None
    dw = torch.empty(d, dtype=ctx.wdtype, device=dev) if need_w else None
    db = torch.empty(d, dtype=ctx.wdtype, device=dev) if need_b else None
    x, n, inner, so, si = _rows(x)
    dy, _, dinner, dso, dsi = _rows(dy)
    mean = stats.data_ptr()
    head = _lib._LAYER_NORM_HEAD.pack(
        _lib.row_dtype_code(x.dtype), _lib.row_dtype_code(ctx.wdtype), n, d, ctx.eps, x.data_ptr(), inner, so, si, _ptr(weight), 0, 0,
        mean, mean + 4 * n, dy.data_ptr(), dinner, dso, dsi, _ptr(dx), _ptr(dw), _ptr(db))
    lib = _lib.load()
    _lib.call_rows(lib.flk_layer_norm_backward, head, dev, lib.flk_layer_norm_workspace_bytes)
    return dx, dw, db, None


class LayerNormFn(torch.autograd.Function):
    """``layer_norm`` with a backward pass for x, weight and bias."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.eps = eps
        ctx.wdtype = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        if not torch.is_grad_enabled():
            return _backward(ctx, dy)
        with torch.no_grad():  # create_graph=True
            out = _backward(ctx, dy)
        return differentiable_once("layer_norm", out, [t for t in (*ctx.saved_tensors[:2], dy) if t is not None])


def layer_norm(
    x: torch.Tensor,
    weight: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    eps: float = 1e-5,
) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension.

    Parameters
    ----------
    x : (..., D) tensor in float32, bfloat16 or float16; rows may be strided (the heads of a packed projection)
    weight, bias : (D,) tensors of one type, x's or float32; either may be missing
    eps : added to the variance, which is the mean of the squared centred values

    Statistics and sums are kept in float32; the result is dense and has x's type.  Differentiable once with respect to
    x, weight and bias, in reverse mode only (no tangents, no ``torch.func``).  Runs on the current stream of x's device, and may be captured into a CUDA graph (a backward pass, as
    torch has it for every operator, only while no graph of the same leaves that was built outside of the capture is alive).
    """
    refuse_tangents("layer_norm", x, weight, bias)
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"x must be a torch.Tensor, not {type(x).__name__}")
    _lib.row_dtype_code(x.dtype)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must have a last dimension of at least one value")
    d = x.shape[-1]
    if d > 1 << 24:
        raise NotImplementedError("rows of more than 2^24 values are not implemented")
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        raise ValueError("eps must be finite and not negative")
    if x.device.type != "cuda":
        _require_cuda(None)
        raise ValueError(f"x must be on a CUDA device (found {x.device})")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, not {type(t).__name__}")
        if t.shape != (d,):
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {(d,)}")
        if t.dtype != x.dtype and t.dtype != torch.float32:
            raise TypeError(f"{name} must be {x.dtype} or float32, not {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"All operands must be on the same device ({name} is on {t.device}, expected {x.device})")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must have one type")
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return LayerNormFn.apply(x, weight, bias, eps)
    return _forward(x, weight, bias, eps, False)[0]
