"""Attention between two ragged sets of rows of the same events on torch CUDA tensors: the queries of an event (its
hits, or a few object queries) read the keys and values of the same event in another batch (its condensates, or all
hits).  There is no counterpart in HGCalML's ``modules``; batches are ragged as everywhere there, rows of all events
behind each other with ``row_splits [E+1]``."""
from __future__ import annotations

from typing import Optional

import torch

from . import _capi as C

_TYPES = (torch.float32, torch.float16, torch.bfloat16)
_MAX_DIM = 128


def _rows(t: torch.Tensor) -> torch.Tensor:
    """The tensor, or a dense copy where its rows have no layout that the kernels read: columns next to each other, every
    row and head in its own place (views of a joint projection are read where they lie)."""
    if t.stride(2) == 1 and all(t.stride(d) > 0 or t.shape[d] == 1 for d in (0, 1)):
        return t
    return t.contiguous()


def _prepare(queries, keys, values, query_row_splits, key_row_splits, scale, key_mask):
    C.require_cuda(queries, keys, values)
    C.refuse_tangents("CrossAttention", queries, keys, values)
    q, k, v = queries, keys, values
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.shape[2] != k.shape[2]:
        raise C.HgcError("CrossAttention expects queries [N, heads, D] and keys and values [M, key heads, D], not "
                         f"{tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    if q.shape[1] < 1 or k.shape[1] < 1 or q.shape[1] % k.shape[1] != 0:
        raise C.HgcError(f"CrossAttention: {k.shape[1]} key heads cannot be shared evenly by {q.shape[1]} heads")
    if not 1 <= q.shape[2] <= _MAX_DIM:
        raise C.HgcError(f"CrossAttention takes heads of 1 to {_MAX_DIM} columns, not {q.shape[2]}")
    if q.dtype not in _TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise C.HgcError("CrossAttention expects queries, keys and values of one type, float32, float16 or bfloat16, not "
                         f"{q.dtype}, {k.dtype} and {v.dtype}")
    if k.device != q.device or v.device != q.device:
        raise C.HgcError("CrossAttention: queries, keys and values live on different devices")
    rs_q, rs_k = C.i32(query_row_splits, q.device), C.i32(key_row_splits, q.device)
    if rs_q.dim() != 1 or rs_k.shape != rs_q.shape or rs_q.shape[0] < 1:
        raise C.HgcError("CrossAttention expects two row splits of equal length, one entry more than there are events")
    if key_mask is not None:
        if key_mask.dtype not in (torch.bool, torch.uint8) or key_mask.numel() != k.shape[0]:
            raise C.HgcError(f"CrossAttention: key_mask must hold one truth value for each of the {k.shape[0]} keys")
        if key_mask.device != q.device:
            raise C.HgcError(f"CrossAttention: key_mask lives on {key_mask.device}, the queries on {q.device}")
        key_mask = key_mask.reshape(-1).contiguous()
    scale = q.shape[2] ** -0.5 if scale is None else float(scale)
    if not 0. < scale < 3.4e38:
        raise C.HgcError(f"CrossAttention: scale must be positive and finite, not {scale}")
    C.check_device(q)
    return _rows(q), _rows(k), _rows(v), rs_q, rs_k, scale, key_mask


def _forward(q, k, v, rs_q, rs_k, scale, mask, with_rest=False):
    out, rest, lse, ws, rc = C.native.cross_attention(q, k, v, rs_q, rs_k, mask, scale, with_rest)
    C.check(rc, "CrossAttention")
    C.check_status(ws)
    return out, rest, lse


def CrossAttentionGrad(grad, queries, keys, values, out, lse, query_row_splits, key_row_splits, scale=None, key_mask=None,
                       need_queries=True, need_keys=True, out_rest=None):
    """Gradients ``(queries, keys, values)`` of ``CrossAttention`` (None for what is not needed; those of keys and values
    come together).  ``out`` and ``lse`` are the forward pass's.  ``out_rest``: what is left of the rows in 16 bits when
    they are rounded, of their type, if known; it makes up for their rounding where few keys have all the weight."""
    q, k, v, rs_q, rs_k, scale, mask = _prepare(queries, keys, values, query_row_splits, key_row_splits, scale, key_mask)
    C.require_cuda(grad, out, lse)
    C.refuse_tangents("CrossAttentionGrad", grad, out, lse)
    if grad.shape != q.shape or out.shape != q.shape or lse.shape != q.shape[:2]:
        raise C.HgcError("CrossAttentionGrad expects grad and out like the queries and one lse per row and head")
    if out.dtype != q.dtype or lse.dtype != torch.float32 or any(t.device != q.device for t in (grad, out, lse)):
        raise C.HgcError("CrossAttentionGrad expects out and lse as CrossAttention returned them, and grad beside them")
    if out_rest is not None:
        C.require_cuda(out_rest)
        if out_rest.shape != out.shape or out_rest.dtype != out.dtype or out_rest.device != out.device:
            raise C.HgcError("CrossAttentionGrad expects out_rest like out")
        out_rest = out_rest.contiguous()
    dq, dk, dv, ws, rc = C.native.cross_attention_grad(grad.to(q.dtype).contiguous(), q, k, v, out.contiguous(), out_rest, lse.contiguous(),
                                                       rs_q, rs_k, mask, scale, need_queries, need_keys)
    C.check(rc, "CrossAttentionGrad")
    C.check_status(ws)
    return dq, dk, dv


class _CrossAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, rs_q, rs_k, scale, mask):
        out, rest, lse = _forward(q, k, v, rs_q, rs_k, scale, mask, with_rest=ctx.needs_input_grad[0] or ctx.needs_input_grad[1])
        ctx.save_for_backward(q, k, v, out, rest, lse, rs_q, rs_k, mask)
        ctx.scale = scale
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)  # no zeros for the logarithms
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _grad_lse):
        if grad is None:
            return (None,) * 7
        q, k, v, out, rest, lse, rs_q, rs_k, mask = ctx.saved_tensors
        need_q, need_k, need_v = ctx.needs_input_grad[:3]
        dq, dk, dv = CrossAttentionGrad(grad, q, k, v, out, lse, rs_q, rs_k, ctx.scale, mask, need_q, need_k or need_v, rest)
        return dq, dk if need_k else None, dv if need_v else None, None, None, None, None


def CrossAttention(queries, keys, values, query_row_splits, key_row_splits, scale: Optional[float] = None, key_mask=None,
                   with_lse: bool = False):
    """``softmax(scale * q.k) v`` over the keys of the query's event.

    ``queries [N, heads, D]``, ``keys`` and ``values [M, key heads, D]`` of one type (float32, float16, bfloat16; D up to
    128), rows and heads at any distance; the heads are shared evenly among the key heads, head h reads key head
    ``h // (heads // key_heads)``.  ``query_row_splits`` and ``key_row_splits [E+1]``: the rows of every event, which may be
    none, and which may end before the tensors do; they ascend from zero (checked with HGC_CHECK_STATUS=1 in the
    environment).  ``scale`` is ``D ** -0.5`` unless given.  ``key_mask [M]`` (bool): keys that no query may see are False, and
    what their rows hold does not matter.  A query that sees no key gets zeros.  Rows that are seen are finite; a NaN among
    them stays one in all that it is a term of.

    Returns the rows ``[N, heads, D]``, with ``with_lse`` also the float32 logarithm of every row's sum of
    exponentials ``[N, heads]`` (``-inf`` without keys), from which results over parts of the keys can be joined.
    Differentiable in queries, keys and values, once and backwards only, with results that do not change from run to run.
    The logarithms carry no gradient: what is joined with them is for use without one."""
    q, k, v, rs_q, rs_k, scale, mask = _prepare(queries, keys, values, query_row_splits, key_row_splits, scale, key_mask)
    # a trace needs a node that stands for the call
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad) or torch.jit.is_tracing():
        out, lse = _CrossAttentionFunction.apply(q, k, v, rs_q, rs_k, scale, mask)
    else:
        out, _, lse = _forward(q, k, v, rs_q, rs_k, scale, mask)
    return (out, lse) if with_lse else out
