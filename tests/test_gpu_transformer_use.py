"""The transformer's operators as a program puts them together: gradients in place of what they are made from, one tensor in several roles, refusals inside a capture, and all of
them in one graph of tensors."""
import math

import numpy as np
import pytest
import torch

from helpers import RTOL_FRO
from test_gpu_transformer import close, down, ops, randn, up  # noqa: F401  (ops is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(1, 768), (7, 64), (300, 768), (1024, 1024), (1030, 2049), (3, 8192), (3, 8193), (20, 20001)], ids=str)
@pytest.mark.parametrize("where", ["dy", "x"])
@pytest.mark.parametrize("accumulate", [0, 1])
def test_layer_norm_gradient_in_place(ops, shape, where, accumulate):  # noqa: F811
    """grad_X written over dY, or over X: the same bits as beside them."""
    from tenmo_amd import _transformer as T

    rows, n = shape
    x, w, b, dy = up(ops, randn(1, rows, n)), up(ops, randn(2, n)), up(ops, randn(3, n)), up(ops, randn(4, rows, n))
    y, mean, rstd = ops.N.layer_norm(x, w, b)
    L = T.load()
    size = L.tenmo_hip_layer_norm_backward_workspace_bytes(rows, n)
    workspace = torch.empty((size + 3) // 4, device="cuda")
    got = []
    for aside in (True, False):
        xs, dys = x.storage.clone(), dy.storage.clone()
        place = dys if where == "dy" else xs
        gx = place.clone() if aside else place
        gw, gb = torch.ones(n, device="cuda"), torch.ones(n, device="cuda")
        torch.cuda.synchronize()
        X = ops.NDBuffer(xs, shape)
        ops.lib.check(L.tenmo_hip_layer_norm_backward_f32(T.view(X), T.address(w), T.address(mean), T.address(rstd), dys.data_ptr(), gx.data_ptr(), gw.data_ptr(), gb.data_ptr(),
                                                          accumulate, workspace.data_ptr(), size, 1))
        got.append((gx, gw, gb))
    # few rows: dw and db are summed in another order beside them than in place, 16 rows against 4 a workgroup
    assert torch.equal(got[0][0], got[1][0])
    for a, c in zip(got[0][1:], got[1][1:]):
        close(a.cpu(), c.cpu(), RTOL_FRO)


@pytest.mark.parametrize("shape", [(5, 64), (300, 768), (9, 2049), (3, 20001)], ids=str)
def test_layer_norm_in_place(ops, shape):  # noqa: F811
    from tenmo_amd import _transformer as T

    x, w = up(ops, randn(5, *shape)), up(ops, randn(6, shape[1]))
    want = down(ops.N.layer_norm(x, w, None)[0])
    ops.lib.check(T.load().tenmo_hip_layer_norm_forward_f32(T.view(x), T.address(w), None, 1e-5, x.data_ptr(), None, None, 1))
    assert torch.equal(down(x), want)


def test_refusals_inside_a_capture(ops):  # noqa: F811
    """A program that catches a refusal while it captures goes on with its graph."""
    N = ops.NDBuffer
    q, wide, x, h, w = up(ops, randn(1, 1, 40, 2, 32)), N.empty((1, 8, 2, 129)), up(ops, randn(2, 6, 64)), up(ops, randn(3, 5, 32)), up(ops, randn(4, 32, 50))
    target, lse, many = torch.arange(5, device="cuda"), N.empty((1, 2, 8)), N.empty((1 << 23, 1))
    words = N(torch.zeros(1, device="cuda"), (32, (1 << 22) + 1), (0, 0))
    calls = [lambda: ops.A.attention(wide, wide, wide), lambda: ops.A.attention_backward(wide, wide, wide, wide, lse, wide),
             lambda: ops.N.layer_norm(x, eps=-1.0), lambda: ops.N.layer_norm_backward(N(x.storage, (2, 0)), None, N.empty((0,)), N.empty((0,)), N.empty((2, 0))),
             lambda: ops.V.vocabulary_loss(many, N.empty((1, 4)), None, torch.zeros(1 << 23, dtype=torch.int64, device="cuda")),
             lambda: ops.V.vocabulary_loss(h, words, None, target),
             lambda: ops.V.vocabulary_loss_backward(h, w, None, target, loss, torch.ones(1, device="cuda"), label_smoothing=2.0)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss = ops.V.vocabulary_loss(h, w, None, target)
        want = down(ops.A.attention(q, q, q, causal=True)[0])
    for call in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(ops.lib.TenmoHipError):
                call()
            o, _ = ops.A.attention(q, q, q, causal=True)
        for _ in range(3):
            o.storage.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(down(o), want)


def grad(t):
    return t.grad().reshape(-1)


@pytest.mark.parametrize("rows", [1, 300])
def test_one_tensor_in_several_roles(ops, rows):  # noqa: F811
    """The gradient of a tensor with several roles in a node is the sum of those it would have in each."""
    T, n = ops.Tensor, 320
    x, w, b = (randn(i, *s).numpy() for i, s in enumerate(((rows, n), (n,), (n,))))
    new = lambda a: T.from_numpy(a, requires_grad=True)  # noqa: E731

    def norm(X, W, B):
        layer = ops.N.LayerNorm(n)
        layer.weight, layer.bias = W, B
        layer(X).backward()

    X, W, B = new(x), new(w), new(w)
    norm(X, W, B)
    X2, W2 = new(x), new(w)
    norm(X2, W2, W2)
    assert np.array_equal(grad(X), grad(X2))
    close(grad(W2), grad(W).astype(np.float64) + grad(B), RTOL_FRO, "weight and bias")
    A, W, B = new(w), new(w), new(b)
    norm(A, W, B)
    A2, B2 = new(w), new(b)
    norm(A2, A2, B2)
    close(grad(A2), grad(A).astype(np.float64) + grad(W), RTOL_FRO, "input and weight")

    h = randn(7, n, n).numpy() * 0.05
    target = (torch.arange(n, device="cuda") * 7) % n
    H, V = new(h), new(h)
    ops.V.VocabularyLoss.forward(H, V, None, target).backward()
    H2 = new(h)
    ops.V.VocabularyLoss.forward(H2, H2, None, target).backward()
    close(grad(H2), grad(H).astype(np.float64) + grad(V), RTOL_FRO, "hidden states and weight")
