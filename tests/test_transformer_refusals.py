"""What the operators of include/tenmo_hip_transformer.h refuse, with the status and message they give; and that header, library and binding
agree.  No GPU: arguments are checked before the device is touched."""
import ctypes as C
import os
import re
import subprocess

import pytest

from tenmo_amd import _lib, _transformer

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHAPE, ARGUMENT, UNSUPPORTED, UNINITIALISED = -2, -3, -5, -1
P = 4096  # a pointer that nothing follows


def view(shape, strides=None, data=P):
    if strides is None:
        strides, n = [], 1
        for s in reversed(shape):
            strides.insert(0, n)
            n *= s
    return C.byref(_lib.make_view(data, 0, shape, strides))


def refused(status, text, rc):
    message = _lib.load().tenmo_hip_last_error().decode()
    assert rc == status and text in message, (rc, message)


def test_header_library_and_binding_agree(tmp_path):
    header = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "tenmo_hip_transformer.h")).read(), flags=re.S)
    declared = {m.group(1): m.group(2).count(",") + 1 for m in re.finditer(r"\b(tenmo_hip_\w+)\s*\(([^;]*?)\)\s*;", header, re.S)}
    assert declared == {name: len(args) for name, (_, args) in _transformer.SIGNATURES.items()}
    _transformer.load()
    src = tmp_path / "t.c"
    src.write_text('#include "tenmo_hip_transformer.h"\nint main(void) { return 0; }\n')
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "include"), "-c", str(src), "-o", str(tmp_path / "t.o")], check=True)


def norm_forward(X=None, eps=1e-5, out=P, mean=P, rstd=P):
    return _transformer.load().tenmo_hip_layer_norm_forward_f32(X or view((4, 8)), P, P, eps, out, mean, rstd, 0)


def test_layer_norm_refusals():
    refused(SHAPE, "rank 0", norm_forward(view(())))
    refused(SHAPE, "last axis is empty", norm_forward(view((3, 0))))
    refused(SHAPE, "negative dimension", norm_forward(view((-3, 4), (4, 1))))
    refused(ARGUMENT, "X has no data", norm_forward(view((3, 4), data=None)))
    refused(ARGUMENT, "eps", norm_forward(eps=-1.0))
    refused(ARGUMENT, "eps", norm_forward(eps=float("nan")))
    refused(ARGUMENT, "null out", norm_forward(out=None))
    refused(ARGUMENT, "mean and rstd", norm_forward(mean=None))
    refused(UNSUPPORTED, "2^27", norm_forward(view((2, (1 << 27) + 1))))
    L = _transformer.load()
    refused(ARGUMENT, "null X", L.tenmo_hip_layer_norm_forward_f32(None, P, P, 1e-5, P, P, P, 0))
    refused(ARGUMENT, "null pointer", L.tenmo_hip_layer_norm_backward_f32(view((4, 8)), P, None, P, P, P, P, P, 0, P, 1 << 20, 0))


def attn_forward(q=(2, 3, 4, 16), k=(2, 5, 2, 16), v=None, scale=0.25, out=P, **kw):
    return _transformer.load().tenmo_hip_attention_forward_f32(kw.get("Q") or view(q), view(k), view(v or k), scale, 0, None, None, out, P, P, 0, 0)


def test_attention_refusals():
    refused(SHAPE, "Q has rank 3", attn_forward(q=(2, 3, 64)))
    refused(SHAPE, "differ", attn_forward(k=(3, 5, 2, 16)))
    refused(SHAPE, "differ", attn_forward(k=(2, 5, 2, 8)))
    refused(SHAPE, "axis 1 of V", attn_forward(v=(2, 6, 2, 16)))
    refused(SHAPE, "multiple", attn_forward(k=(2, 5, 3, 16)))
    refused(SHAPE, "multiple", attn_forward(k=(2, 5, 0, 16)))
    refused(UNSUPPORTED, "head size 129", attn_forward(q=(2, 3, 4, 129), k=(2, 5, 2, 129)))
    refused(UNSUPPORTED, "head size 0", attn_forward(q=(2, 3, 4, 0), k=(2, 5, 2, 0)))
    refused(UNSUPPORTED, "2^25", attn_forward(q=(1 << 15, 1 << 15, 4, 16), k=(1 << 15, 5, 2, 16)))
    refused(UNSUPPORTED, "2^20", attn_forward(q=(1 << 19, 1, 4, 16), k=(1 << 19, 5, 2, 16)))
    refused(UNSUPPORTED, "2^27", attn_forward(q=(1, 1, 4, 16), k=(1, 1 << 28, 2, 16)))
    refused(ARGUMENT, "scale", attn_forward(scale=float("inf")))
    refused(ARGUMENT, "null out", attn_forward(out=None))
    L = _transformer.load()

    def backward(gq=(2, 3, 4, 16), gk=None, strides=None, out=P):
        return L.tenmo_hip_attention_backward_f32(view((2, 3, 4, 16)), view((2, 5, 2, 16)), view((2, 5, 2, 16)), 0.25, 0, None, None, out, P, P,
                                                  view(gq, strides), None if gk is None else view(gk), None, 0, P, 1 << 20, 0)

    refused(SHAPE, "axis 1 of grad_Q", backward(gq=(2, 5, 4, 16)))
    refused(SHAPE, "axis 2 of grad_K", backward(gk=(2, 5, 4, 16)))
    refused(ARGUMENT, "stride of 0", backward(strides=(192, 0, 16, 1)))
    refused(ARGUMENT, "null out, lse or dOut", backward(out=None))
    refused(SHAPE, "multiple", L.tenmo_hip_attention_forward_workspace_bytes(1, 1, 1, 3, 2, 16))
    refused(SHAPE, "multiple", L.tenmo_hip_attention_backward_workspace_bytes(-1, 1, 1, 2, 2, 16))
    refused(UNSUPPORTED, "2^28", L.tenmo_hip_attention_backward_workspace_bytes(1, 8, (1 << 22) + 1, 64, 8, 16))


def test_vocabulary_loss_refusals():
    L = _transformer.load()

    def forward(h=(4, 8), w=(8, 10), target=P, smoothing=0.0, lse=P):
        return L.tenmo_hip_vocabulary_loss_forward_f32(view(h), view(w), None, target, 1, -100, smoothing, P, lse, P, P, P, 0, 0)

    def backward(gw=(8, 10), strides=None, reduction=2, valid=P, upstream=P):
        return L.tenmo_hip_vocabulary_loss_backward_f32(view((4, 8)), view((8, 10)), None, P, 1, -100, 0.0, P, upstream, reduction, valid, P, view(gw, strides), None, 0, P, 0, 0)

    refused(SHAPE, "H has rank 3", forward(h=(2, 2, 8)))
    refused(SHAPE, "inner dims", forward(w=(7, 10)))
    refused(SHAPE, "vocabulary >= 1", forward(w=(8, 0)))
    refused(UNSUPPORTED, "words", forward(w=(8, (1 << 22) + 1)))
    refused(UNSUPPORTED, "2^38", forward(h=(1 << 20, 8), w=(8, 1 << 20)))
    refused(ARGUMENT, "label_smoothing", forward(smoothing=1.5))
    refused(ARGUMENT, "label_smoothing", forward(smoothing=float("nan")))
    refused(ARGUMENT, "null pointer", forward(target=None))
    refused(ARGUMENT, "null pointer", forward(lse=None))
    refused(SHAPE, "axis 1 of grad_W", backward(gw=(8, 11)))
    refused(ARGUMENT, "stride of 0", backward(strides=(0, 1)))
    refused(ARGUMENT, "reduction", backward(reduction=3))
    refused(ARGUMENT, "valid_count", backward(valid=None))
    refused(ARGUMENT, "null pointer", backward(upstream=None))
    refused(SHAPE, "tokens", L.tenmo_hip_vocabulary_loss_forward_workspace_bytes(-1, 8, 10))
    refused(SHAPE, "dimension", L.tenmo_hip_vocabulary_loss_backward_workspace_bytes(4, 0, 10))


def test_calls_without_initialisation_fail_cleanly():
    L = _transformer.load()
    if L.tenmo_hip_get_stream():
        pytest.skip("library already initialised in this process")
    refused(UNINITIALISED, "not initialised", norm_forward())
    refused(UNINITIALISED, "not initialised", attn_forward())
    refused(UNINITIALISED, "not initialised", L.tenmo_hip_vocabulary_loss_forward_f32(view((4, 8)), view((8, 10)), None, P, 1, -100, 0.0, P, P, P, P, P, 0, 0))
    refused(UNINITIALISED, "not initialised", L.tenmo_hip_attention_forward_workspace_bytes(1, 1, 1, 1, 1, 16))


def test_layer_norm_workspace_refusals():
    bytes_of = _transformer.load().tenmo_hip_layer_norm_backward_workspace_bytes
    refused(SHAPE, "columns >= 1", bytes_of(4, 0))
    refused(SHAPE, "rows >= 0", bytes_of(-1, 8))
    refused(UNSUPPORTED, "2^27", bytes_of(2, (1 << 27) + 1))
    assert bytes_of(0, 8) == 0 and bytes_of(4, 8) > 0
