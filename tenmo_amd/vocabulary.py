"""Cross-entropy over a vocabulary from the hidden states, without the logits: ``vocabulary_loss`` / ``vocabulary_loss_backward`` on buffers,
``VocabularyLoss`` on tensors.  The arithmetic is the library's (``tenmo_hip_vocabulary_loss_*``, include/tenmo_hip_transformer.h).

h is [tokens, dim], w [dim, vocabulary] (a ``Linear``'s weight, or the transposed view of an embedding it is tied to).
"""
from __future__ import annotations

import math
from typing import List, NamedTuple, Optional, Tuple

import torch

from . import _transformer as _t
from ._lib import TenmoHipError, check
from .ndbuffer import NDBuffer
from .tensor import Tensor

REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}  # the cross-entropy kernels' own encoding


class Loss(NamedTuple):
    per_sample: NDBuffer       # [tokens], 0 where the target is ignore_index
    lse: NDBuffer              # [tokens], for the backward call
    loss_sum: NDBuffer         # [1]
    valid_count: torch.Tensor  # int32 [1] on the device: the mean is loss_sum / max(valid_count, 1)


def _sizes(h: NDBuffer, w: NDBuffer, bias: Optional[NDBuffer]):
    if h.rank() != 2 or w.rank() != 2 or h.shape[1] != w.shape[0]:
        raise TenmoHipError(-2, f"vocabulary_loss: hidden states {h.shape} and weight {w.shape}: [tokens, dim] and [dim, vocabulary] are needed")
    _t.dense(bias, (w.shape[1],), "vocabulary_loss: bias")
    return h.shape[0], h.shape[1], w.shape[1]


def vocabulary_loss(h: NDBuffer, w: NDBuffer, bias: Optional[NDBuffer], target: torch.Tensor, ignore_index: int = -100, label_smoothing: float = 0.0,
                    sync: bool = False) -> Loss:
    """target: int64 or int32 [tokens] on the device; one outside the vocabulary that is not ignore_index gives NaN."""
    sizes = m, _, _ = _sizes(h, w, bias)
    t = _t.device_ints(target, m, "vocabulary_loss: target", (torch.int64, torch.int32))
    L, joined = _t.enter(h, w, bias)
    try:
        loss = Loss(_t.empty(h, m), _t.empty(h, m), _t.empty(h, 1), torch.empty(1, dtype=torch.int32, device=h.storage.device))
        _, ws, size = _keep = _t.workspace(h, L.tenmo_hip_vocabulary_loss_forward_workspace_bytes(*sizes))
        check(L.tenmo_hip_vocabulary_loss_forward_f32(_t.view(h), _t.view(w), _t.address(bias), t, 1 if target.dtype == torch.int64 else 0,
                                                      ignore_index, label_smoothing, loss.per_sample.data_ptr(), loss.lse.data_ptr(), loss.loss_sum.data_ptr(),
                                                      loss.valid_count.data_ptr(), ws, size, 1 if sync else 0))
    finally:
        _t.leave(joined)
    return loss


def vocabulary_loss_backward(h: NDBuffer, w: NDBuffer, bias: Optional[NDBuffer], target: torch.Tensor, loss: Loss, upstream: torch.Tensor, reduction: str = "mean",
                             ignore_index: int = -100, label_smoothing: float = 0.0, need: Tuple[bool, bool, bool] = (True, True, True), into=None,
                             sync: bool = False) -> Tuple[Optional[NDBuffer], Optional[NDBuffer], Optional[NDBuffer]]:
    """(grad_h, grad_w, grad_bias) for the gradient ``upstream`` of the reduced loss (fp32 on the device: [tokens] for "none", else one value); those not
    needed, and grad_bias without a bias, are None.  grad_w lies in memory in the order of w: the gradient of a transposed view is the transposed view of a
    dense one.  ``into``: three buffers (grad_h and grad_bias dense, grad_w with any strides) or None each, which are added to instead."""
    sizes = m, d, v = _sizes(h, w, bias)
    t = _t.device_ints(target, m, "vocabulary_loss_backward: target", (torch.int64, torch.int32))
    if reduction not in REDUCTIONS:
        raise TenmoHipError(-3, f"vocabulary_loss_backward: reduction must be one of {sorted(REDUCTIONS)}, got {reduction!r}")
    up = _t.device_ints(upstream, m if reduction == "none" else 1, "vocabulary_loss_backward: upstream", (torch.float32,))
    _t.dense(loss.lse, (m,), "vocabulary_loss_backward: lse")
    if into is not None:
        _t.dense(into[0], (m, d), "vocabulary_loss_backward: grad_h")
        _t.dense(into[2], (v,), "vocabulary_loss_backward: grad_bias")
    L, joined = _t.enter(h, w, bias, *(into or ()))
    try:
        if into is not None:
            gh, gw, gb = into
        else:
            gh = _t.empty(h, m, d) if need[0] else None
            gb = _t.empty(h, v) if need[2] and bias is not None else None
            gw = None
            if need[1]:
                gw = _t.empty(w, v, d).transpose() if w.strides[0] == 1 and d > 1 else _t.empty(w, d, v)
        _, ws, size = _keep = _t.workspace(h, L.tenmo_hip_vocabulary_loss_backward_workspace_bytes(*sizes))
        check(L.tenmo_hip_vocabulary_loss_backward_f32(_t.view(h), _t.view(w), _t.address(bias), t, 1 if target.dtype == torch.int64 else 0,
                                                       ignore_index, label_smoothing, loss.lse.data_ptr(), up, REDUCTIONS[reduction], loss.valid_count.data_ptr(),
                                                       _t.address(gh), _t.view(gw), _t.address(gb), 0 if into is None else 1,
                                                       ws, size, 1 if sync else 0))
    finally:
        _t.leave(joined)
    return gh, gw, gb


def _rows(h: NDBuffer) -> NDBuffer:
    """[..., dim] as [tokens, dim]."""
    if h.rank() < 3:
        return h
    if not h.is_contiguous():
        raise TenmoHipError(-5, f"VocabularyLoss: hidden states {h.shape} with strides {h.strides}: more than two axes need to be dense")
    return h.view((math.prod(h.shape[:-1]), h.shape[-1]), (h.shape[-1], 1), h.offset)


class VocabularyLoss:
    """The loss at a language model's head in the autograd graph."""

    @staticmethod
    def forward(h: Tensor, w: Tensor, bias: Optional[Tensor], target: torch.Tensor, reduction: str = "mean", ignore_index: int = -100,
                label_smoothing: float = 0.0, track_grad: bool = True, sync: bool = False, tied: bool = False) -> Tensor:
        """h: [..., dim], as the layers before it return it, and target as many values.  w: [dim, vocabulary], or, ``tied``, an embedding [vocabulary, dim], whose gradient it is then that
        is added to (a ``Tensor.transpose`` is a leaf of its own).  The loss is [1], or of h's leading axes for "none"."""
        if reduction not in REDUCTIONS:
            raise TenmoHipError(-3, f"VocabularyLoss: reduction must be one of {sorted(REDUCTIONS)}, got {reduction!r}")
        parents = (h, w) + ((bias,) if bias is not None else ())
        kind = dict(ignore_index=ignore_index, label_smoothing=label_smoothing)
        b = bias.buffer if bias is not None else None
        if tied and w.rank() != 2:
            raise TenmoHipError(-2, f"VocabularyLoss: an embedding is [vocabulary, dim], got {w.shape()}")
        rows, weight = _rows(h.buffer), w.buffer.transpose() if tied else w.buffer
        loss = vocabulary_loss(rows, weight, b, target, sync=sync, **kind)
        if reduction == "none":
            out = Tensor(NDBuffer(loss.per_sample.storage, h.shape()[:-1]))
        elif reduction == "sum":
            out = Tensor(loss.loss_sum)
        else:
            out = Tensor(NDBuffer(loss.loss_sum.storage / loss.valid_count.clamp(min=1), (1,)))
        if track_grad and any(p.requires_grad for p in parents):
            def backward(output: Tensor, retain_graph: bool = False) -> List[Tensor]:
                upstream = output.gradbox.storage[:output.numels()]

                def add(into):
                    gh, gw, gb = into
                    gh = None if gh is None else NDBuffer(gh.storage, rows.shape)
                    gw = gw.transpose() if tied and gw is not None else gw
                    vocabulary_loss_backward(rows, weight, b, target, loss, upstream, reduction=reduction, into=(gh, gw, gb), **kind)

                got = _t.into_gradients((h, w, bias), add)
                if not retain_graph:
                    output.zero_grad()
                return got

            out.requires_grad = True
            out.add_ancestry(backward, *parents)
        return out
