"""``attention``: the row-normalised product with exp(scores), next to ``fmmv``.

``fmmv`` weighs the rows of ``v`` with ``k(x_i, c_j)``; attention weighs them with ``exp(s_ij)``, normalised over the keys
that a query may see.  As there, the n x m block of weights is never stored: the kernels of ``libfalkon_b200``
(include/falkon_b200.h) form it tile by tile, forward and backward.  There is no CPU path.
"""
import math
from typing import Optional, Tuple, Union

import torch

from .. import _lib
from .fmmv import _require_cuda
from .utils import differentiable_once, refuse_tangents

__all__ = ("attention", "AttentionFn")


def _strided(t: torch.Tensor) -> torch.Tensor:
    """``t``, or a dense copy of it where its layout is none that the kernels read (unit stride over the head dimension,
    16-byte aligned address and strides, no dimension that is broadcast)."""
    sb, sn, sh, sd = t.stride()
    b, n, h, _ = t.shape
    unit = 16 // t.element_size() - 1
    odd = b > 1 and (sb & unit or sb < 1) or n > 1 and (sn & unit or sn < 1) or h > 1 and (sh & unit or sh < 1)
    if sd == 1 and t.data_ptr() & 15 == 0 and not odd:
        return t
    # clone and not contiguous(): a dense tensor whose address is not aligned needs a copy too
    return t.clone(memory_format=torch.contiguous_format)


def _t4(t: torch.Tensor):
    b, n, h, _ = t.stride()
    return t.data_ptr(), b, n, h


def _ptr(t: Optional[torch.Tensor]):
    return 0 if t is None else t.data_ptr()


def _pack(q, k, v, out, out_lo, lse, opts) -> bytes:
    """flk_attention_args up to the gradients' tensors."""
    scale, softcap, causal, slopes, prefix_lens, kv_lens, q_starts, q_docs, k_docs = opts
    b, nq, hq, d = q.shape
    _, nk, hk, _ = k.shape
    # (tables of no entries have no address, and there is nothing for the labels to tell apart)
    qd, qs, kd, ks = (0, 0, 0, 0) if k_docs is None or nq == 0 or nk == 0 else (q_docs.data_ptr(), q_docs.stride(0), k_docs.data_ptr(), k_docs.stride(0))
    return _lib._ATTENTION_FORWARD.pack(
        _lib._ROW_TYPES[q.dtype], b, nq, nk, hq, hk, d, causal, 0, scale, softcap, *_t4(q), *_t4(k), *_t4(v), *_t4(out),
        _ptr(out_lo), _ptr(lse), _ptr(slopes), _ptr(prefix_lens), _ptr(kv_lens), _ptr(q_starts), qd, qs, kd, ks)


_NO_TENSOR = (0, 0, 0, 0)


def _dense_like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _forward(q, k, v, opts, with_lse, with_lo=False):
    lib = _lib.load()
    out = _dense_like(q)
    out_lo = _dense_like(q) if with_lo and q.dtype != torch.float32 else None
    lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32, device=q.device) if with_lse else None
    _lib.call_rows(lib.flk_attention_forward, _pack(q, k, v, out, out_lo, lse, opts) + _lib._ATTENTION_NO_GRADS, q.device,
                   lib.flk_attention_workspace_bytes, 0)
    return out, out_lo, lse


def _backward(ctx, dout, _):
    if dout is None:
        return None, None, None, None
    refuse_tangents("attention", dout)
    q, k, v, out, out_lo, lse, *kept = ctx.saved_tensors
    kept = iter(kept)
    opts = tuple(next(kept) if held else t for t, held in zip(ctx.opts, ctx.held))
    need_q, need_k, need_v, _ = ctx.needs_input_grad
    dq = _dense_like(q) if need_q else None
    dk = dv = None
    if need_k or need_v:
        dk, dv = _dense_like(k), _dense_like(v)
    lib = _lib.load()
    dout = _strided(dout)
    grads = _lib._ATTENTION_GRADS.pack(*_t4(dout), *(_NO_TENSOR if dq is None else _t4(dq)),
                                       *(_NO_TENSOR if dk is None else _t4(dk)), *(_NO_TENSOR if dv is None else _t4(dv)))
    head = _pack(q, k, v, out, out_lo, lse, opts) + grads
    _lib.call_rows(lib.flk_attention_backward, head, q.device, lib.flk_attention_workspace_bytes, 1)
    return dq, dk if need_k else None, dv if need_v else None, None


class AttentionFn(torch.autograd.Function):
    """``attention`` with a backward pass for q, k and v (the log-sum-exp that it also returns passes no gradient).  With
    16-bit data it also keeps what rounding took from ``out``, as large as ``out``: the backward pass subtracts
    ``dout . out`` from every weight's gradient, and the rounding would be the largest error of dq and dk."""

    @staticmethod
    def forward(ctx, q, k, v, opts):
        out, out_lo, lse = _forward(q, k, v, opts, True, True)
        ctx.save_for_backward(q, k, v, out, out_lo, lse, *(t for t in opts if isinstance(t, torch.Tensor)))
        ctx.opts = tuple(None if isinstance(t, torch.Tensor) else t for t in opts)
        ctx.held = tuple(isinstance(t, torch.Tensor) for t in opts)
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    def backward(ctx, *grads):
        if not torch.is_grad_enabled():
            return _backward(ctx, *grads)
        with torch.no_grad():  # create_graph=True
            out = _backward(ctx, *grads)
        return differentiable_once("attention", out, [*ctx.saved_tensors[:3], *(g for g in grads if g is not None)])


def _table(name: str, t: Optional[torch.Tensor], shape, device, labels: bool = False) -> Optional[torch.Tensor]:
    """An integer table on the data's device, as int32 with unit stride over its last dimension.  Numbers beyond int32 become
    its ends; labels, which must not fall together, become negative, that is padding (2^31 wraps)."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, not {type(t).__name__}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.device != device:
        raise ValueError(f"All operands must be on the same device ({name} is on {t.device}, expected {device})")
    if t.dtype != torch.int32:
        if t.dtype != torch.int64:
            raise TypeError(f"{name} must be int32 or int64, not {t.dtype}")
        t = t.clamp(-(2**31), 2**31 if labels else 2**31 - 1).to(torch.int32)
    return t if t.dim() == 0 or t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _left_out(opts, nq: int, nk: int) -> torch.Tensor:
    """The distance, per sequence, that the kernels leave out of every score (include/falkon_b200.h)."""
    kv_lens, q_starts = opts[5], opts[6].clamp(-(2**29), 2**29)
    last = max(nk, 1) - 1 if kv_lens is None else kv_lens.clamp(1, max(nk, 1)) - 1
    return (q_starts - q_starts.clamp(min=-nq).clamp(max=last)).abs()


def _refuse(q, k, v):
    """Says what is wrong with operands that do not fit."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, not {type(t).__name__}")
        if t.dim() != 4:
            raise ValueError(f"{name} must be 4-D (batch, rows, heads, head dimension), found {t.dim()}-D")
    _lib.row_dtype_code(q.dtype)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"Data types of q, k and v must be equal (found {q.dtype}, {k.dtype}, {v.dtype})")
    b, _, hq, d = q.shape
    hk = k.shape[2]
    if k.shape[0] != b or k.shape[3] != d or v.shape != k.shape:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit together")
    if d < 1 or d > 128:
        raise NotImplementedError(f"head dimension {d}: 1 to 128 are implemented")
    if hk < 1 or hq < 1 or hq % hk != 0:
        raise ValueError(f"{hq} query heads cannot share {hk} key heads")
    _require_cuda(None)
    raise ValueError(f"q, k and v must be on one CUDA device (found {q.device}, {k.device}, {v.device})")


def attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    causal: bool = False,
    scale: Optional[float] = None,
    softcap: Optional[float] = None,
    slopes: Optional[torch.Tensor] = None,
    prefix_lens: Optional[torch.Tensor] = None,
    documents: Optional[torch.Tensor] = None,
    q_documents: Optional[torch.Tensor] = None,
    kv_lens: Optional[torch.Tensor] = None,
    q_starts: Optional[torch.Tensor] = None,
    return_lse: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``out[b, i, h] = sum_j softmax_j(s_ij) v[b, j, h']`` over the keys j that query i may see.

    ``s_ij = softcap * tanh(scale * q_i . k_j / softcap) - slopes[h] * |p_i - j|`` with ``p_i`` the query's position.

    Parameters
    ----------
    q : (B, Nq, Hq, D) tensor in float32, bfloat16 or float16, D <= 128
    k, v : (B, Nk, Hk, D) tensors of the same type; Hq is a multiple of Hk and consecutive query heads share a key head
    causal : query i sees keys up to its own position only
    scale : factor of the dot products, default ``1 / sqrt(D)``
    softcap : scores are bounded by a tanh to (-softcap, softcap); None or 0: they are not
    slopes : (Hq,) float32, the distance bias of each query head (a constant: it gets no gradient)
    prefix_lens : (B,) integers; with ``causal``, the first keys of a sequence that every query may see
    documents : (B, Nk) integers; a query sees the keys of its own document only.  A negative label marks padding, which
        sees and shows nothing, and so does one of 2^31 and more
    q_documents : (B, Nq) integers, the queries' documents; default ``documents`` where Nq == Nk
    kv_lens : (B,) integers; keys at or behind this length do not exist (a cache's length), default Nk
    q_starts : (B,) integers, position of the first query of a sequence; by default the last query stands at the last
        key, that is at ``kv_lens - Nq``.  A right-padded batch of Nq == Nk rows takes zeros here
    return_lse : also return ``log sum_j exp(s_ij)``, (B, Hq, Nq) float32 (without gradient)

    A query that sees no key gets zeros, and -inf in the log-sum-exp.  What such queries, padding rows, keys behind
    ``kv_lens`` and, with ``causal``, keys that no query reaches hold does not matter, NaN included.  Integer tables are
    read on the device: lengths beyond [0, Nk] count as the nearer end.  At most 65535 sequences, 65535 heads, 2^29 rows.
    Differentiable once with respect to q, k and v, in reverse mode only (no tangents, no ``torch.func``).  Runs on the current stream of the data's device, allocates its output
    and workspace from torch's allocator, and may be captured into a CUDA graph (a backward pass, as torch has it for every
    operator, only while no graph of the same leaves that was built outside of the capture is alive).  With 16-bit data every wait
    inside a kernel is bounded: rows that a stalled GPU does not finish within a second are NaN, and so are their gradients.
    """
    refuse_tangents("attention", q, k, v, slopes)
    try:
        fits = q.dtype is k.dtype is v.dtype and q.dtype in _lib._ROW_TYPES and k.shape == v.shape and q.device == k.device == v.device
        b, nq, hq, d = q.shape
        kb, nk, hk, kd = k.shape
        fits = fits and kb == b and kd == d and 1 <= d <= 128 and hk >= 1 and hq >= 1 and hq % hk == 0 and q.device.type == "cuda"
    except (AttributeError, ValueError, TypeError):
        fits = False
    if not fits:
        _refuse(q, k, v)
    dev = q.device
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    softcap = 0.0 if softcap is None else float(softcap)
    if not math.isfinite(scale) or not (0.0 <= softcap < math.inf):
        raise ValueError("scale must be finite, softcap finite and not negative")
    if slopes is not None:
        if not isinstance(slopes, torch.Tensor) or slopes.dtype != torch.float32 or slopes.shape != (hq,) or slopes.device != dev:
            raise ValueError(f"slopes must be a float32 tensor of {hq} entries on {dev}")
        if slopes.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("slopes are constants: their gradient is not implemented")
        slopes = slopes.contiguous()
    if prefix_lens is not None and not causal:
        raise ValueError("prefix_lens needs causal=True: without it every query sees all keys anyway")
    if q_documents is not None and documents is None:
        raise ValueError("q_documents needs documents")
    if documents is not None and q_documents is None:
        if nq != nk:
            raise ValueError("q_documents must be given where queries and keys differ in number")
        q_documents = documents
    opts = (scale, softcap, 1 if causal else 0, slopes, _table("prefix_lens", prefix_lens, (b,), dev),
            _table("kv_lens", kv_lens, (b,), dev), _table("q_starts", q_starts, (b,), dev),
            _table("q_documents", q_documents, (b, nq), dev, True), _table("documents", documents, (b, nk), dev, True))
    pad = -d % 8
    if pad:  # the kernels read whole vectors of 16 bytes; zeros change no dot product
        q, k, v = (torch.nn.functional.pad(t, (0, pad)) for t in (q, k, v))
    q, k, v = _strided(q), _strided(k), _strided(v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse = AttentionFn.apply(q, k, v, opts)
    else:
        out, _, lse = _forward(q, k, v, opts, return_lse)
    if pad:
        out = out[..., :d]
    if not return_lse:
        return out
    if slopes is not None and q_starts is not None:
        lse = lse - slopes[:, None] * _left_out(opts, nq, nk)[:, None, None]
    return out, lse
