"""ctypes binding of include/tenmo_hip_transformer.h, and what its operators share: results and workspaces in torch's allocator, and
their order with the caller's stream.

The library enqueues on one stream (``tenmo_hip_get_stream``).  An operator called under another current torch stream joins the two: the
library's stream waits for the current one before the launch, the current one for the library's behind it.  Under
``torch.cuda.graph`` that makes the launches part of the captured graph.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Callable, Optional, Sequence

import torch

from . import _lib
from ._lib import TenmoHipError, check
from .ndbuffer import NDBuffer

_vp, _ptr, _i64, _i32, _f32 = C.POINTER(_lib.CView), C.c_void_p, C.c_int64, C.c_int32, C.c_float

# name -> (restype, argtypes); every function include/tenmo_hip_transformer.h declares
SIGNATURES = {
    "tenmo_hip_layer_norm_forward_f32": (C.c_int, [_vp, _ptr, _ptr, _f32, _ptr, _ptr, _ptr, _i32]),
    "tenmo_hip_layer_norm_backward_workspace_bytes": (_i64, [_i64, _i64]),
    "tenmo_hip_layer_norm_backward_f32": (C.c_int, [_vp, _ptr, _ptr, _ptr, _ptr, _ptr, _ptr, _ptr, _i32, _ptr, _i64, _i32]),
    "tenmo_hip_attention_forward_workspace_bytes": (_i64, [_i64] * 6),
    "tenmo_hip_attention_forward_f32": (C.c_int, [_vp, _vp, _vp, _f32, _i32, _ptr, _ptr, _ptr, _ptr, _ptr, _i64, _i32]),
    "tenmo_hip_attention_backward_workspace_bytes": (_i64, [_i64] * 6),
    "tenmo_hip_attention_backward_f32": (C.c_int, [_vp, _vp, _vp, _f32, _i32, _ptr, _ptr, _ptr, _ptr, _ptr, _vp, _vp, _vp, _i32, _ptr, _i64, _i32]),
    "tenmo_hip_vocabulary_loss_forward_workspace_bytes": (_i64, [_i64] * 3),
    "tenmo_hip_vocabulary_loss_forward_f32": (C.c_int, [_vp, _vp, _ptr, _ptr, _i32, _i64, _f32, _ptr, _ptr, _ptr, _ptr, _ptr, _i64, _i32]),
    "tenmo_hip_vocabulary_loss_backward_workspace_bytes": (_i64, [_i64] * 3),
    "tenmo_hip_vocabulary_loss_backward_f32": (C.c_int, [_vp, _vp, _ptr, _ptr, _i32, _i64, _f32, _ptr, _ptr, _i32, _ptr, _ptr, _vp, _ptr, _i32, _ptr, _i64, _i32]),
}

_bound = None


def load() -> C.CDLL:
    """The library with these functions bound (raises if one is missing)."""
    global _bound
    L = _lib.load()
    if _bound is not L:
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        L.hipStreamGetFlags.argtypes = [_ptr, C.POINTER(C.c_uint)]
        _bound = L
    return L


def enter(*operands: Optional[NDBuffer]):
    """(library, token): the library initialised, every operand on its device, its stream behind the current one.  ``leave(token)`` puts the
    current stream behind the library's, and has to follow also where the call between them raises: a capture cannot end while the library's stream is forked from it."""
    _lib.init()
    for b in operands:
        if b is not None and b.storage.get_device() != 0:  # _lib.init's device
            raise TenmoHipError(-3, f"operand on {b.storage.device}: the library runs on device 0")
    L = _bound or load()
    current, own = _current_stream(0), L.tenmo_hip_get_stream() or 0
    if current == own or (current == 0 and _follows_default(L, own)):
        return L, None
    stream, library = torch.cuda.current_stream(0), torch.cuda.ExternalStream(own, device=0)
    library.wait_stream(stream)
    return L, (stream, library)


def leave(token) -> None:
    if token is not None:
        current, library = token
        current.wait_stream(library)


_current_stream = torch._C._cuda_getCurrentRawStream


def _follows_default(L: C.CDLL, stream: int) -> bool:
    """Whether the stream is ordered with the default stream by itself (it was not created as a non-blocking one)."""
    flags = C.c_uint(1)
    return L.hipStreamGetFlags(stream, C.byref(flags)) == 0 and flags.value == 0


def empty(like: NDBuffer, *shape: int) -> NDBuffer:
    n = 1
    strides = []
    for s in reversed(shape):
        strides.append(n)
        n *= s
    b = NDBuffer.__new__(NDBuffer)  # (what the constructor checks holds here)
    b.storage = like.storage.new_empty(n or 1)
    b.shape, b.strides, b.offset = shape, tuple(reversed(strides)), 0
    return b


_VIEW = [struct.Struct(f"@Pqi4x{rank}q{8 * (_lib.MAX_RANK - rank)}x{rank}q{8 * (_lib.MAX_RANK - rank)}x") for rank in range(_lib.MAX_RANK + 1)]


def view(b: Optional[NDBuffer]):
    """Of a buffer, as the library takes it."""
    if b is None:
        return None
    rank = len(b.shape)
    if rank > _lib.MAX_RANK:
        raise TenmoHipError(-2, f"rank {rank} exceeds max_rank {_lib.MAX_RANK}")
    return C.byref(_lib.CView.from_buffer_copy(_VIEW[rank].pack(b.storage.data_ptr(), b.offset, rank, *b.shape, *b.strides)))


def workspace(like: NDBuffer, nbytes: int):
    """(tensor that owns it, address, bytes); torch's allocator aligns to 512 bytes and, under capture, keeps it for the graph."""
    check(nbytes)
    if nbytes == 0:
        return None, None, 0
    t = like.storage.new_empty((nbytes + 3) // 4)
    return t, t.data_ptr(), nbytes


def address(b: Optional[NDBuffer]) -> Optional[int]:
    """Of a dense buffer's first element."""
    return None if b is None else b.storage.data_ptr() + 4 * b.offset


def dense(b: Optional[NDBuffer], shape: tuple, what: str) -> None:
    if b is not None and (b.shape != shape or not (b.strides == (1,) or b.is_contiguous())):
        raise TenmoHipError(-2, f"{what} must be dense with shape {shape}, got shape {b.shape} with strides {b.strides}")


def into_gradients(tensors: Sequence, call: Callable) -> list:
    """For the tensors of a node (None where it has none): ``call(into)`` with the gradients that are to be added to, None where there is none; once for each role where a tensor has
    several, since two gradients of one call may not share a place.  The tensors that got one."""
    wanted = [t is not None and t.requires_grad for t in tensors]
    given = [id(t) for t in tensors if t is not None]
    if len(set(given)) == len(given):
        call([t.ensure_gradbox() if w else None for t, w in zip(tensors, wanted)])
    else:
        for role, w in enumerate(wanted):
            if w:
                call([t.ensure_gradbox() if i == role else None for i, t in enumerate(tensors)])
    return [t for t, w in zip(tensors, wanted) if w]


def device_ints(t: Optional[torch.Tensor], n: int, what: str, dtypes=(torch.int32,)) -> Optional[int]:
    """Address of a dense device tensor of n whole numbers."""
    if t is None:
        return None
    if t.dtype not in dtypes or t.numel() != n or not t.is_contiguous() or not t.is_cuda or t.get_device() != 0:
        raise TenmoHipError(-3, f"{what}: needs {n} dense {' or '.join(str(d) for d in dtypes)} values on the library's device, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()
