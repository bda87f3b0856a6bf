"""The transformer's operators as a program puts them together: gradients in place of what they are made from, one tensor in several roles, refusals inside a capture, and all of
them in one graph of tensors."""
import math

import numpy as np
import pytest
import torch

from helpers import RTOL_FRO
from test_gpu_transformer import block_tensors, close, down, ops, randn, up  # noqa: F401  (ops is a fixture)

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


def test_a_block_and_its_head_in_one_graph(ops):  # noqa: F811
    """norm -> joint projection -> attention -> norm -> loss over a tied embedding: one backward call from the loss to every leaf, against 64-bit autograd."""
    h, norm, qkv, head_norm, emb, target, H = block_tensors(ops)
    B, S, E = h.shape()
    target[5::11] = -100
    y = head_norm(ops.A.Attention.packed(qkv(norm(h)), heads=H, causal=True))
    loss = ops.V.VocabularyLoss.forward(y, emb, None, target.reshape(B, S), tied=True)
    loss.backward()
    tensors = [h, norm.weight, norm.bias, qkv.weight, qkv.bias, head_norm.weight, head_norm.bias, emb]
    x, nw, nb, w, b, hw, hb, e = leaves = [torch.from_numpy(t.to_numpy()).double().requires_grad_(True) for t in tensors]
    q, k, v = (torch.nn.functional.layer_norm(x, (E,), nw, nb, 1e-5) @ w + b).reshape(B, S, 3, H, E // H).permute(2, 0, 3, 1, 4)
    s = (q @ k.transpose(2, 3) / math.sqrt(E // H)).masked_fill(torch.ones(S, S).triu(1).bool(), -math.inf)
    o = torch.nn.functional.layer_norm((torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B * S, E), (E,), hw, hb, 1e-5)
    want = torch.nn.functional.cross_entropy(o @ e.t(), target.cpu())
    want.backward()
    close(loss.to_numpy(), want.detach().reshape(1), RTOL_FRO, "loss")
    names = ("h", "norm.weight", "norm.bias", "qkv.weight", "qkv.bias", "head_norm.weight", "head_norm.bias", "embedding")
    for t, ref, what in zip(tensors, leaves, names):  # four operators in a row, each with a gradient's tolerance of its own
        close(t.grad(), ref.grad.numpy(), 8 * RTOL_FRO, what)


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_vocabulary_loss_of_a_batch(ops, reduction, tied, bias):  # noqa: F811
    """Hidden states [batch, length, dim] and an embedding give what [tokens, dim] and its transposed view do, the gradient in the embedding's own place."""
    T, B, S, d, v = ops.Tensor, 3, 30, 48, 700
    h, e, b = randn(1, B, S, d).numpy(), randn(2, v, d).numpy(), randn(3, v).numpy()
    target = torch.randint(0, v, (B, S), generator=torch.Generator().manual_seed(4)).cuda()
    target[1, 3:9] = -100
    new = lambda a: T.from_numpy(np.ascontiguousarray(a), requires_grad=True)  # noqa: E731
    H, W, C = new(h), new(e if tied else e.T), new(b) if bias else None
    got = ops.V.VocabularyLoss.forward(H, W, C, target, reduction=reduction, tied=tied)
    got.backward()
    H2, W2, C2 = new(h.reshape(B * S, d)), new(e).transpose() if tied else new(e.T), new(b) if bias else None
    want = ops.V.VocabularyLoss.forward(H2, W2, C2, target.reshape(-1), reduction=reduction)
    want.backward()
    assert got.shape() == ((B, S) if reduction == "none" else (1,)) and H.grad().shape == (B, S, d)
    assert np.array_equal(got.to_numpy().reshape(-1), want.to_numpy().reshape(-1)) and np.array_equal(grad(H), grad(H2))
    assert not bias or np.array_equal(C.grad(), C2.grad())
    # (the gradient of the view lies along the other axis: the same sums by other tiles)
    close(W.grad().T if tied else W.grad(), W2.grad(), RTOL_FRO, "grad_w")


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("v", [7, 3000])
def test_vocabulary_loss_of_no_tokens(ops, reduction, tied, v):  # noqa: F811
    """Nothing to learn from: a loss of zero and gradients of zero, which leave what is added to as it is."""
    N, d = ops.NDBuffer, 40
    h, b, w = N.empty((0, d)), up(ops, randn(1, v)), up(ops, randn(2, v, d)).transpose() if tied else up(ops, randn(2, d, v))
    target = torch.zeros(0, dtype=torch.int64, device="cuda")
    loss = ops.V.vocabulary_loss(h, w, b, target)
    assert down(loss.loss_sum) == 0.0 and int(loss.valid_count) == 0
    upstream = torch.ones(0 if reduction == "none" else 1, device="cuda")
    gh, gw, gb = ops.V.vocabulary_loss_backward(h, w, b, target, loss, upstream, reduction=reduction)
    assert gh.shape == (0, d) and gw.shape == (d, v) and not down(gw).any() and not down(gb).any()
    want = randn(3, d, v)
    gw, gb = up(ops, want.t().contiguous()).transpose() if tied else up(ops, want), up(ops, randn(4, v))
    ops.V.vocabulary_loss_backward(h, w, b, target, loss, upstream, reduction=reduction, into=(None, gw, gb))
    assert torch.equal(down(gw), want) and torch.equal(down(gb), randn(4, v))


def test_vocabulary_loss_of_a_batch_refusals(ops):  # noqa: F811
    T, N = ops.Tensor, ops.NDBuffer
    w, t = T.zeros(48, 700), torch.zeros(60, dtype=torch.int64, device="cuda")
    cases = [(T(N.zeros((2, 48, 30)).transpose()), w, False, "dense"), (T.zeros(2, 31, 48), w, False, "60"), (T.zeros(2, 30, 48), w, True, "inner|needed"), (T.zeros(2, 30, 48), T.zeros(48), True, "embedding")]
    for h, weight, tied, text in cases:
        with pytest.raises(ops.lib.TenmoHipError, match=text if text != "60" else "needs 62"):
            ops.V.VocabularyLoss.forward(h, weight, None, t, tied=tied)
