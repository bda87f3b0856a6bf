"""Attention: ``attention`` / ``attention_backward`` on buffers, ``Attention`` on tensors.  The arithmetic is the library's
(``tenmo_hip_attention_*``, include/tenmo_hip_transformer.h).

q is [batch, queries, heads, dim], k and v [batch, keys, kv_heads, dim], with any strides: slices of one projection [batch, queries, 3 * heads * dim]
need no copy, and the result reshapes to [batch, queries, heads * dim] for the next one.
"""
from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple

import torch

from . import _transformer as _t
from ._lib import TenmoHipError, check
from .ndbuffer import NDBuffer
from .tensor import Tensor


def _sizes(q: NDBuffer, k: NDBuffer, v: NDBuffer):
    for b, what in ((q, "q"), (k, "k"), (v, "v")):
        if b.rank() != 4:
            raise TenmoHipError(-2, f"attention: {what} must be [batch, length, heads, dim], got {b.shape}")
    return q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3]


def attention(q: NDBuffer, k: NDBuffer, v: NDBuffer, scale: Optional[float] = None, causal: bool = False, key_lengths: Optional[torch.Tensor] = None,
              query_starts: Optional[torch.Tensor] = None, statistics: bool = True, sync: bool = False) -> Tuple[NDBuffer, Optional[NDBuffer]]:
    """(out, lse): softmax(scale * q . k^T) . v over the allowed keys, and the logarithm of each row's sum [batch, heads, queries] for the
    backward call (None without ``statistics``).  scale: 1 / sqrt(dim) by default.  Sequence b has key_lengths[b] keys (device int32; all of them by
    default); with ``causal`` query i sees the keys up to position query_starts[b] + i (device int32; the last positions by default)."""
    sizes = _sizes(q, k, v)
    batch, queries, _, heads, _, dim = sizes
    lengths = _t.device_ints(key_lengths, batch, "attention: key_lengths")
    starts = _t.device_ints(query_starts, batch, "attention: query_starts")
    L, joined = _t.enter(q, k, v)
    try:
        out = _t.empty(q, batch, queries, heads, dim)
        lse = _t.empty(q, batch, heads, queries) if statistics else None
        _, ws, size = _keep = _t.workspace(q, L.tenmo_hip_attention_forward_workspace_bytes(*sizes))
        check(L.tenmo_hip_attention_forward_f32(_t.view(q), _t.view(k), _t.view(v), 1.0 / math.sqrt(dim) if scale is None else scale,
                                                1 if causal else 0, lengths, starts, out.data_ptr(), _t.address(lse), ws, size, 1 if sync else 0))
    finally:
        _t.leave(joined)
    return out, lse


def attention_backward(q: NDBuffer, k: NDBuffer, v: NDBuffer, out: NDBuffer, lse: NDBuffer, dout: NDBuffer, scale: Optional[float] = None, causal: bool = False,
                       key_lengths: Optional[torch.Tensor] = None, query_starts: Optional[torch.Tensor] = None, need: Sequence[bool] = (True, True, True),
                       into: Optional[Sequence[Optional[NDBuffer]]] = None, sync: bool = False) -> Tuple[Optional[NDBuffer], Optional[NDBuffer], Optional[NDBuffer]]:
    """(grad_q, grad_k, grad_v) for the upstream gradient dout (dense, out's shape), with out and lse of the forward call and its other
    arguments; those not needed are None.  ``into``: three buffers of the shapes of q, k and v (any strides, no two elements of the three at one place) or None each, which are
    added to instead."""
    sizes = _sizes(q, k, v)
    batch, queries, _, heads, _, dim = sizes
    lengths = _t.device_ints(key_lengths, batch, "attention_backward: key_lengths")
    starts = _t.device_ints(query_starts, batch, "attention_backward: query_starts")
    _t.dense(out, q.shape, "attention_backward: out")
    _t.dense(dout, q.shape, "attention_backward: dout")
    _t.dense(lse, (batch, heads, queries), "attention_backward: lse")
    L, joined = _t.enter(q, k, v, out, lse, dout, *(into or ()))
    try:
        grads = tuple(into) if into is not None else tuple(_t.empty(b, *b.shape) if n else None for b, n in zip((q, k, v), need))
        _, ws, size = _keep = _t.workspace(q, L.tenmo_hip_attention_backward_workspace_bytes(*sizes))
        views = [_t.view(g) for g in grads]
        check(L.tenmo_hip_attention_backward_f32(_t.view(q), _t.view(k), _t.view(v), 1.0 / math.sqrt(dim) if scale is None else scale,
                                                 1 if causal else 0, lengths, starts, _t.address(out), _t.address(lse), _t.address(dout), *views,
                                                 0 if into is None else 1, ws, size, 1 if sync else 0))
    finally:
        _t.leave(joined)
    return grads


def packed_views(qkv: NDBuffer, heads: int, kv_heads: Optional[int] = None) -> Tuple[NDBuffer, NDBuffer, NDBuffer]:
    """q, k and v in a projection [batch, length, (heads + 2 * kv_heads) * dim], as views."""
    kv_heads = heads if kv_heads is None else kv_heads
    if qkv.rank() != 3 or heads < 1 or kv_heads < 1 or qkv.shape[2] % (heads + 2 * kv_heads):
        raise TenmoHipError(-2, f"packed_views: {qkv.shape} does not hold {heads} query heads and {kv_heads} key and value heads")
    (b, n, width), (sb, sn, sw) = qkv.shape, qkv.strides
    dim = width // (heads + 2 * kv_heads)
    return tuple(qkv.view((b, n, h, dim), (sb, sn, dim * sw, sw), qkv.offset + first * dim * sw)
                 for h, first in ((heads, 0), (kv_heads, heads), (kv_heads, heads + kv_heads)))


class Attention:
    """Attention in the autograd graph."""

    @staticmethod
    def forward(q: Tensor, k: Tensor, v: Tensor, scale: Optional[float] = None, causal: bool = False, key_lengths: Optional[torch.Tensor] = None,
                query_starts: Optional[torch.Tensor] = None, track_grad: bool = True, sync: bool = False) -> Tensor:
        mask = dict(scale=scale, causal=causal, key_lengths=key_lengths, query_starts=query_starts)
        track = track_grad and (q.requires_grad or k.requires_grad or v.requires_grad)
        o, lse = attention(q.buffer, k.buffer, v.buffer, statistics=track, sync=sync, **mask)
        out = Tensor(o)
        if track:
            def backward(output: Tensor, retain_graph: bool = False) -> List[Tensor]:
                got = _t.into_gradients((q, k, v), lambda into: attention_backward(q.buffer, k.buffer, v.buffer, o, lse, output.gradbox, into=into, **mask))
                if not retain_graph:
                    output.zero_grad()
                return got

            out.requires_grad = True
            out.add_ancestry(backward, q, k, v)
        return out

    @staticmethod
    def packed(qkv: Tensor, heads: int, kv_heads: Optional[int] = None, scale: Optional[float] = None, causal: bool = False,
               key_lengths: Optional[torch.Tensor] = None, query_starts: Optional[torch.Tensor] = None, track_grad: bool = True, sync: bool = False) -> Tensor:
        """Of a joint projection [batch, length, (heads + 2 * kv_heads) * dim]; the result is [batch, length, heads * dim].  Nothing is copied either
        way: the gradients are added to the projection's gradient in place."""
        mask = dict(scale=scale, causal=causal, key_lengths=key_lengths, query_starts=query_starts)
        track = track_grad and qkv.requires_grad
        views = packed_views(qkv.buffer, heads, kv_heads)
        o, lse = attention(*views, statistics=track, sync=sync, **mask)
        out = Tensor(NDBuffer(o.storage, (o.shape[0], o.shape[1], o.shape[2] * o.shape[3])))
        if track:
            def backward(output: Tensor, retain_graph: bool = False) -> List[Tensor]:
                dout = NDBuffer(output.gradbox.storage, o.shape)
                attention_backward(*views, o, lse, dout, into=packed_views(qkv.ensure_gradbox(), heads, kv_heads), **mask)
                if not retain_graph:
                    output.zero_grad()
                return [qkv]

            out.requires_grad = True
            out.add_ancestry(backward, qkv)
        return out
