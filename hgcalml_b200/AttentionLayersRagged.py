"""A torch layer on ``NormRotate`` and ``CrossAttention``: the rows of an event read those of a second ragged batch of the same
events, as an object query reads hits, or a hit the condensates of its event.  HGCalML's ``modules`` have no such layer; inputs
are lists with ``row_splits`` as those of its GravNet layers, and the dense layers are the ones these use."""
from __future__ import annotations

import torch

from . import _capi as C
from .cross_attention_op import CrossAttention
from .GravNetLayersRagged import _Dense
from .norm_rotate_op import NormRotate


class RaggedCrossAttention(torch.nn.Module):
    """Inputs ``[x [N, n_in], context [M, n_context], row_splits [E+1], context_row_splits [E+1]]``; returns ``[N, n_out]``.

    ``n_heads`` heads of ``n_head_features`` columns, which share ``n_key_heads`` key heads; queries and keys are scaled to unit
    size per head and, where positions are given (coordinates ``[N, axes]`` or integers ``[N]``, as ``NormRotate`` takes them),
    turned by them.  ``key_mask [M]``: rows of the context that nobody may see are False, and what they and their positions hold
    does not matter.  A row without any gets what the output transform makes of zeros.  Rows behind the last event get the same;
    where gradients are asked for they have to be finite, as the rows of any dense layer.

    The context is projected to keys and values at once; ``prepare`` does that ahead of time, for a context that many
    queries are asked of one after the other, and its result may be passed in place of the context."""

    def __init__(self, n_heads: int, n_head_features: int, n_out: int, n_in: int, n_context: int, n_key_heads: int = 0,
                 rotary_dim=None, base: float = 10000., interleaved: bool = False, activation=None):
        super().__init__()
        n_key_heads = n_key_heads or n_heads
        if n_heads < 1 or n_key_heads < 1 or n_heads % n_key_heads != 0:
            raise ValueError(f"{n_key_heads} key heads cannot be shared evenly by {n_heads} heads")
        self.n_heads, self.n_key_heads, self.n_head_features = n_heads, n_key_heads, n_head_features
        self.how = dict(rotary_dim=rotary_dim, base=base, interleaved=interleaved)
        self.query_transform = _Dense(n_in, n_heads * n_head_features, None)
        self.context_transform = _Dense(n_context, 2 * n_key_heads * n_head_features, None)
        self.query_scale = torch.nn.Parameter(torch.ones(n_head_features))
        self.key_scale = torch.nn.Parameter(torch.ones(n_head_features))
        self.output_transform = _Dense(n_heads * n_head_features, n_out, activation)

    @staticmethod
    def _seen(key_mask, context, key_positions):
        """Zeros where nobody looks: a gradient of zero does not make up for a row of NaN in the gradients of the transforms."""
        if key_mask is None or not torch.is_grad_enabled():
            return context, key_positions
        hidden = key_mask.reshape(-1) == 0

        def clear(t):  # the ops refuse what does not fit
            fits = t is not None and t.dim() > 0 and t.shape[0] == hidden.shape[0] and t.device == hidden.device
            return t.masked_fill(hidden.reshape(-1, *[1] * (t.dim() - 1)), 0) if fits else t

        return clear(context), clear(key_positions)

    def _keys_values(self, context):
        both = self.context_transform(context).unflatten(-1, (2, self.n_key_heads, self.n_head_features))
        return both[:, 0], both[:, 1]

    def prepare(self, context, key_positions=None, key_mask=None):
        """Keys, scaled and turned, and values of a context.  ``key_mask`` is needed where gradients are and masked rows may hold
        anything."""
        context, key_positions = self._seen(key_mask, context, key_positions)
        keys, values = self._keys_values(context)
        keys, _ = NormRotate(keys, None, self.key_scale, None, key_positions, **self.how)
        return keys, values

    def forward(self, inputs, query_positions=None, key_positions=None, key_mask=None):
        x, context, row_splits, context_row_splits = inputs
        queries = self.query_transform(x).unflatten(-1, (self.n_heads, self.n_head_features))
        if isinstance(context, tuple):
            if key_positions is not None:
                raise C.HgcError("RaggedCrossAttention: the positions of a context are given where it is prepared")
            keys, values = context
            queries, _ = NormRotate(queries, None, self.query_scale, None, query_positions, **self.how)
        else:
            context, key_positions = self._seen(key_mask, context, key_positions)
            keys, values = self._keys_values(context)
            queries, keys = NormRotate(queries, keys, self.query_scale, self.key_scale, query_positions, key_positions, **self.how)
        out = CrossAttention(queries, keys, values, row_splits, context_row_splits, key_mask=key_mask)
        return self.output_transform(out.flatten(1))
