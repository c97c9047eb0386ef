"""Norm of the heads of queries and keys and their rotation by positions, on torch CUDA tensors: what prepares the
two sets of rows for ``CrossAttention``.  There is no counterpart in HGCalML's ``modules``; positions are the hits'
coordinates, one or several axes of them, or integers."""
from __future__ import annotations

from typing import Optional

import torch

from . import _capi as C

_TYPES = (torch.float32, torch.float16, torch.bfloat16)
_POSITION_TYPES = (torch.float32, torch.int32, torch.int64)
_MAX_DIM = 128


def _rows(t):
    """As it lies, or a dense copy where columns do not lie next to each other."""
    return t if t is None or t.stride(2) == 1 else t.contiguous()


def _check_set(what, x, weight, positions, like):
    if x.dim() != 3 or x.dtype != like.dtype or x.shape[2] != like.shape[2] or x.device != like.device:
        raise C.HgcError(f"NormRotate expects {what} [N, heads, D], of one type and width and on one device with the queries")
    if x.shape[1] < 1:
        raise C.HgcError(f"NormRotate: {what} have no heads")
    if weight is not None:
        C.require_cuda(weight)
        if weight.shape != (x.shape[2],) or weight.dtype not in (torch.float32, x.dtype) or weight.device != x.device:
            raise C.HgcError(f"NormRotate expects the weight of the {what} as {x.shape[2]} values of their type or float32 beside them")
    if positions is not None:
        C.require_cuda(positions)
        if positions.dim() not in (1, 2) or positions.shape[0] != x.shape[0] or positions.device != x.device:
            raise C.HgcError(f"NormRotate expects positions [N] or [N, axes] beside the {what}, not {tuple(positions.shape)}")
        if positions.dtype not in _POSITION_TYPES:
            raise C.HgcError(f"NormRotate takes positions in float32, int32 or int64, not {positions.dtype}")
        if positions.requires_grad and torch.is_grad_enabled():
            raise C.HgcError("NormRotate has no gradient for positions: detach them")


def _prepare(queries, keys, query_weight, key_weight, query_positions, key_positions, rotary_dim, base, eps):
    C.require_cuda(queries, keys)
    C.refuse_tangents("NormRotate", queries, keys, query_weight, key_weight, query_positions, key_positions)
    if queries.dim() != 3 or queries.dtype not in _TYPES or not 1 <= queries.shape[2] <= _MAX_DIM:
        raise C.HgcError(f"NormRotate expects queries [N, heads, D] in float32, float16 or bfloat16 with D from 1 to {_MAX_DIM}, not "
                         f"{tuple(queries.shape)} in {queries.dtype}")
    _check_set("queries", queries, query_weight, query_positions, queries)
    if keys is None:
        if key_weight is not None or key_positions is not None:
            raise C.HgcError("NormRotate: a weight or positions for keys that are not there")
    else:
        _check_set("keys", keys, key_weight, key_positions, queries)
    given = [p for p in (query_positions, key_positions) if p is not None]
    axes = 1
    if given:
        axes = given[0].shape[1] if given[0].dim() == 2 else 1
        if any(p.dtype != given[0].dtype or (p.shape[1] if p.dim() == 2 else 1) != axes for p in given):
            raise C.HgcError("NormRotate expects positions of queries and keys of one type, with equally many axes")
    if axes < 1:
        raise C.HgcError("NormRotate: positions without axes")
    dim = queries.shape[2]
    rotary = dim // (2 * axes) * 2 * axes if rotary_dim is None else int(rotary_dim)
    if rotary < 0 or rotary > dim or rotary % (2 * axes) != 0:
        raise C.HgcError(f"NormRotate: {rotary} columns of {dim} cannot turn in pairs of {axes} axes")
    if not 1. < base < 1e30 or not 0. <= eps < float("inf"):
        raise C.HgcError("NormRotate expects a base above one and an eps of at least zero")
    C.check_device(queries)
    flat = [None if p is None else p.detach().contiguous() for p in (query_positions, key_positions)]
    weights = [None if w is None else w.contiguous() for w in (query_weight, key_weight)]
    return _rows(queries), _rows(keys), *weights, *flat, rotary, axes


def _forward(q, k, wq, wk, pq, pk, rotary, axes, interleaved, base, eps):
    yq, yk, rc = C.native.norm_rotate(q, k, wq, wk, pq, pk, rotary, axes, interleaved, base, eps)
    C.check(rc, "NormRotate")
    return yq, yk


class _NormRotateFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, pq, pk, rotary, axes, interleaved, base, eps):
        ctx.save_for_backward(q, k, wq, wk, pq, pk)
        ctx.how = rotary, axes, interleaved, base, eps
        ctx.set_materialize_grads(False)
        return _forward(q, k, wq, wk, pq, pk, rotary, axes, interleaved, base, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_q, grad_k):
        q, k, wq, wk, pq, pk = ctx.saved_tensors
        need = ctx.needs_input_grad
        # a set none of whose gradients is asked for, or whose result was not used, is left out
        use_q, use_k = grad_q is not None and (need[0] or need[2]), grad_k is not None and (need[1] or need[3])
        sets = [(q, wq, pq, grad_q, need[2])] if use_q else []
        if use_k:
            sets.append((k, wk, pk, grad_k, need[3]))
        if not sets:
            return (None,) * 11
        first, second = sets[0], sets[1] if len(sets) > 1 else (None,) * 5
        dense = [None if x[0] is None else x[3].to(q.dtype).contiguous() for x in (first, second)]
        d1, d2, w1, w2, rc = C.native.norm_rotate_grad(dense[0], dense[1], first[0], second[0], first[1], second[1], first[2], second[2],
                                                       bool(first[4]), bool(second[4]), *ctx.how)
        C.check(rc, "NormRotate's gradient")
        dq, dwq = (d1, w1) if use_q else (None, None)
        dk, dwk = ((d2, w2) if use_q else (d1, w1)) if use_k else (None, None)
        return dq if need[0] else None, dk if need[1] else None, dwq, dwk, None, None, None, None, None, None, None


def NormRotate(queries, keys=None, query_weight=None, key_weight=None, query_positions=None, key_positions=None, *,
               rotary_dim: Optional[int] = None, base: float = 10000., interleaved: bool = False, eps: float = 1e-6):
    """Scales every head of ``queries [N, heads, D]`` and of ``keys [M, key heads, D]`` (None: queries alone) to a root mean
    square of one, ``x / sqrt(mean(x^2) + eps) * weight``, and turns it by its row's positions, all in one launch.

    Both sets have one type (float32, float16, bfloat16) and D up to 128; rows and heads may lie at any distance.  Weights
    ``[D]`` are of that type or float32 (None: ones).  Positions ``[N]`` or ``[N, axes]`` are float32 (coordinates),
    int32 or int64, of one type for both sets (None: the set is not turned).  The leading ``rotary_dim`` columns (all that
    fit unless given), in equal parts for the axes, form pairs -- the halves of an axis' part, or neighbouring columns with
    ``interleaved`` -- and pair i turns by ``position / base ** (i / pairs)``.

    Returns ``(queries, keys)`` as dense tensors of the inputs' type (keys None if not given).  Differentiable in rows and
    weights, once and backwards only; positions get no gradient.  Results do not change from run to run."""
    q, k, wq, wk, pq, pk, rotary, axes = _prepare(queries, keys, query_weight, key_weight, query_positions, key_positions, rotary_dim,
                                                  base, eps)
    how = (rotary, axes, bool(interleaved), float(base), float(eps))
    # a trace needs a node that stands for the call
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, wq, wk)) or torch.jit.is_tracing():
        return _NormRotateFunction.apply(q, k, wq, wk, pq, pk, *how)
    return _forward(q, k, wq, wk, pq, pk, *how)
