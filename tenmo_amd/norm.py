"""Layer norm over the last axis: ``layer_norm`` / ``layer_norm_backward`` on buffers, ``LayerNorm`` as a layer beside ``net.Linear``.
The arithmetic is the library's (``tenmo_hip_layer_norm_*``, include/tenmo_hip_transformer.h)."""
from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple

from . import _transformer as _t
from ._lib import TenmoHipError, check
from .ndbuffer import NDBuffer
from .tensor import Tensor


def _rows(x: NDBuffer) -> Tuple[int, int]:
    if x.rank() < 1:
        raise TenmoHipError(-2, "layer_norm: needs at least one axis")
    n = x.shape[-1]
    return math.prod(x.shape[:-1]) if n else 0, n


def layer_norm(x: NDBuffer, weight: Optional[NDBuffer] = None, bias: Optional[NDBuffer] = None, eps: float = 1e-5,
               statistics: bool = True, sync: bool = False) -> Tuple[NDBuffer, Optional[NDBuffer], Optional[NDBuffer]]:
    """(out, mean, rstd) of x, any strides; mean and rstd (one value a row, for the backward call) are None without ``statistics``."""
    rows, n = _rows(x)
    _t.dense(weight, (n,), "layer_norm: weight")
    _t.dense(bias, (n,), "layer_norm: bias")
    L, joined = _t.enter(x, weight, bias)
    try:
        out = _t.empty(x, *x.shape)
        mean, rstd = (_t.empty(x, rows), _t.empty(x, rows)) if statistics else (None, None)
        check(L.tenmo_hip_layer_norm_forward_f32(_t.view(x), _t.address(weight), _t.address(bias), eps, out.data_ptr(),
                                                 _t.address(mean), _t.address(rstd), 1 if sync else 0))
    finally:
        _t.leave(joined)
    return out, mean, rstd


def layer_norm_backward(x: NDBuffer, weight: Optional[NDBuffer], mean: NDBuffer, rstd: NDBuffer, dy: NDBuffer, need_x: bool = True,
                        need_weight: Optional[bool] = None, need_bias: Optional[bool] = None, into: Optional[Sequence[Optional[NDBuffer]]] = None,
                        sync: bool = False) -> Tuple[Optional[NDBuffer], Optional[NDBuffer], Optional[NDBuffer]]:
    """(grad_x, grad_weight, grad_bias) for the upstream gradient dy (dense); those not needed are None (by default the last two when there is
    no weight).  ``into``: three dense buffers or None each, which are added to instead."""
    rows, n = _rows(x)
    _t.dense(weight, (n,), "layer_norm_backward: weight")
    _t.dense(dy, x.shape, "layer_norm_backward: dy")
    _t.dense(mean, (rows,), "layer_norm_backward: mean")
    _t.dense(rstd, (rows,), "layer_norm_backward: rstd")
    need_weight = weight is not None if need_weight is None else need_weight
    need_bias = weight is not None if need_bias is None else need_bias
    if into is not None:
        for g, shape, what in zip(into, (x.shape, (n,), (n,)), ("grad_x", "grad_weight", "grad_bias")):
            _t.dense(g, shape, "layer_norm_backward: " + what)
    L, joined = _t.enter(x, weight, mean, rstd, dy, *(into or ()))
    try:
        gx, gw, gb = into if into is not None else (_t.empty(x, *x.shape) if need_x else None, _t.empty(x, n) if need_weight else None,
                                                    _t.empty(x, n) if need_bias else None)
        _, ws, size = _keep = _t.workspace(x, L.tenmo_hip_layer_norm_backward_workspace_bytes(rows, n) if gw is not None or gb is not None else 0)
        check(L.tenmo_hip_layer_norm_backward_f32(_t.view(x), _t.address(weight), _t.address(mean), _t.address(rstd), _t.address(dy),
                                                  _t.address(gx), _t.address(gw), _t.address(gb), 0 if into is None else 1, ws, size, 1 if sync else 0))
    finally:
        _t.leave(joined)
    return gx, gw, gb


class LayerNorm:
    """A layer with a learned weight and bias over the last axis."""

    def __init__(self, features: int, eps: float = 1e-5):
        self.weight = Tensor.ones(features, requires_grad=True)
        self.bias = Tensor.zeros(features, requires_grad=True)
        self.eps, self.training = eps, True

    def parameters(self) -> List[Tensor]:
        return [self.weight, self.bias]

    def __call__(self, xs: Tensor, sync: bool = False) -> Tensor:
        track = self.training and (xs.requires_grad or self.weight.requires_grad or self.bias.requires_grad)
        y, mean, rstd = layer_norm(xs.buffer, self.weight.buffer, self.bias.buffer, self.eps, statistics=track, sync=sync)
        out = Tensor(y)
        if track:
            w, b = self.weight, self.bias

            def backward(output: Tensor, retain_graph: bool = False) -> List[Tensor]:
                got = _t.into_gradients((xs, w, b), lambda into: layer_norm_backward(xs.buffer, w.buffer, mean, rstd, output.gradbox, into=into))
                if not retain_graph:
                    output.zero_grad()
                return got

            out.requires_grad = True
            out.add_ancestry(backward, xs, w, b)
        return out
