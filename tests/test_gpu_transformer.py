"""Layer norm, attention and the vocabulary loss on the GPU against plain formulas in 64 bits.

Tolerances: relative Frobenius error 1e-5 for results and 2e-5 for gradients, the library's own for products (helpers.RTOL_FRO).  1e-5 is 168
roundings of 2^-24, all in one direction.  The operators' longest chains: a dot product of 128 terms in four accumulators is 32 + 7 roundings of its
terms' magnitudes, an exponential below its row's maximum by t adds t + 2 of its value (t <= 20 where a value counts: e^-20 is below 2^-28), sums over keys
or rows add pairwise or in runs whose roundings have both signs; a gradient has two of these in a row.
"""
import math

import numpy as np
import pytest
import torch

from helpers import RTOL_FRO, rel_fro

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import tenmo_amd.attention as A
    import tenmo_amd.norm as N
    import tenmo_amd.vocabulary as V
    from tenmo_amd import _lib
    from tenmo_amd.ndbuffer import NDBuffer
    from tenmo_amd.tensor import Tensor

    _lib.init(0)

    class NS:
        pass

    NS.A, NS.N, NS.V, NS.lib, NS.NDBuffer, NS.Tensor = A, N, V, _lib, NDBuffer, Tensor
    return NS


def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).float()


def up(ops, t):
    """A host tensor as a buffer of its own: torch's view (shape, strides, offset) over an uploaded copy of its storage."""
    if t is None:
        return None
    base = t.contiguous() if t._base is None else t._base
    if t._base is None:
        t = base
    return ops.NDBuffer(base.reshape(-1).cuda(), tuple(t.shape), tuple(t.stride()), t.storage_offset())


def down(b):
    return b.storage.cpu().as_strided(b.shape, b.strides, b.offset) if b.shape else b.storage.cpu()[b.offset]


def close(got, want, tol, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]), what
    err = rel_fro(got[~inf], want[~inf])
    print(f"{what}: {err:.2e}", flush=True)
    assert err <= tol, (what, err)


# ---- layer norm -----------------------------------------------------------------------------------------------------------------


def norm_reference(x, w, b, eps, dy):
    x, dy = x.double().contiguous().requires_grad_(True), dy.double()
    w, b = ((t.double().requires_grad_(True) if t is not None else None) for t in (w, b))
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    y = (x - mean) * rstd
    y = y * w if w is not None else y
    y = y + b if b is not None else y
    y.backward(dy)
    return [None if t is None else t.detach().numpy() for t in (y, mean[..., 0].reshape(-1), rstd[..., 0].reshape(-1), x.grad, None if w is None else w.grad, None if b is None else b.grad)]


NORM_SHAPES = [(1, 1), (3, 1), (1, 5), (1, 768), (7, 64), (5, 255), (9, 256), (4, 257), (130, 512), (33, 769), (2, 3, 1023), (515, 1024), (6, 1025), (1030, 2049), (3, 4097), (2, 8192),
               (3, 8193), (2, 20001), (1500, 300), (2100, 1000), (1200, 5000), (4099, 33), (1025, 2)]


@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
@pytest.mark.parametrize("affine", [True, False])
def test_layer_norm(ops, shape, affine):
    n = shape[-1]
    x, dy = randn(1, *shape) * 2 + 3, randn(2, *shape)
    w, b = (randn(3, n) + 1, randn(4, n)) if affine else (None, None)
    want = norm_reference(x, w, b, 1e-5, dy)
    X, W, B, DY = (up(ops, t) for t in (x, w, b, dy))
    y, mean, rstd = ops.N.layer_norm(X, W, B, 1e-5)
    gx, gw, gb = ops.N.layer_norm_backward(X, W, mean, rstd, DY)
    # x - mean loses what the mean's size has over the spread's: a factor (3 + 2) / 2 of the roundings
    close(down(y), want[0], RTOL_FRO, "y")
    close(down(mean), want[1], RTOL_FRO, "mean")
    if n > 1:
        close(down(rstd), want[2], RTOL_FRO, "rstd")
    if n > 2:  # of one column nothing is left, of two next to nothing
        close(down(gx), want[3], 2 * RTOL_FRO, "grad_x")
    if affine:
        if n > 1:
            close(down(gw), want[4], 2 * RTOL_FRO, "grad_weight")
        close(down(gb), want[5], 2 * RTOL_FRO, "grad_bias")
        into = [up(ops, randn(9, *s)) for s in (shape, (n,), (n,))]
        before = [down(t).double().numpy() for t in into]
        ops.N.layer_norm_backward(X, W, mean, rstd, DY, into=into)
        for t, g, old in zip(into, (gx, gw, gb), before):
            close(down(t), down(g).double().numpy() + old, 2.0 ** -23, "accumulated")
    y2, none, _ = ops.N.layer_norm(X, W, B, 1e-5, statistics=False)
    assert none is None and torch.equal(down(y2), down(y))


@pytest.mark.parametrize("shape", [(20, 300), (3000, 300), (5, 9000)], ids=str)
def test_layer_norm_one_gradient_at_a_time(ops, shape):
    x, dy, w = up(ops, randn(1, *shape)), up(ops, randn(2, *shape)), up(ops, randn(3, shape[1]))
    y, mean, rstd = ops.N.layer_norm(x, w, w)
    all_of_them = [down(g) for g in ops.N.layer_norm_backward(x, w, mean, rstd, dy)]
    for i in range(3):
        some = ops.N.layer_norm_backward(x, w, mean, rstd, dy, need_x=i == 0, need_weight=i == 1, need_bias=i == 2)
        assert [g is not None for g in some] == [i == j for j in range(3)] and torch.equal(down(some[i]), all_of_them[i])


@pytest.mark.parametrize("view", ["rows", "axes", "columns", "column"])
def test_layer_norm_of_views(ops, view):
    base = randn(5, 12, 10, 40)
    x = {"rows": base[::2, 1:9, 3:36], "axes": base.transpose(0, 1)[:, :, :33], "columns": base[:, :, ::2], "column": base.transpose(1, 2)[:, 1:2, :]}[view]
    assert x._base is not None
    n = x.shape[-1]
    w, b, dy = randn(6, n), randn(7, n), randn(8, *x.shape)
    want = norm_reference(x, w, b, 1e-3, dy)
    X, W, B, DY = up(ops, x), up(ops, w), up(ops, b), up(ops, dy)
    y, mean, rstd = ops.N.layer_norm(X, W, B, 1e-3)
    grads = ops.N.layer_norm_backward(X, W, mean, rstd, DY)
    for got, ref, what in zip((y,) + grads, (want[0],) + tuple(want[3:]), ("y", "grad_x", "grad_weight", "grad_bias")):
        close(down(got), ref, 2 * RTOL_FRO, what)


def test_layer_norm_large_mean_and_constant_rows(ops):
    """Rows far from zero keep their spread (the squares are taken around the mean), and a constant row gives the bias."""
    x = (torch.arange(8 * 96) % 7).float().reshape(8, 96) + 4096.0  # exact in fp32, deviations of 0 .. 6
    x[3] = 5.0
    b = randn(1, 96)
    want = norm_reference(x, None, b, 1e-5, x)
    y, mean, rstd = ops.N.layer_norm(up(ops, x), None, up(ops, b), 1e-5)
    # the mean of 4096 is rounded to 2^-12, against a spread of 2
    close(down(y), want[0], 2.0 ** -12, "y")
    assert np.array_equal(down(y)[3].numpy(), b.numpy())


def test_layer_norm_empty(ops):
    x = ops.NDBuffer.empty((0, 16))
    w = up(ops, randn(1, 16))
    y, mean, rstd = ops.N.layer_norm(x, w, w)
    gx, gw, gb = ops.N.layer_norm_backward(x, w, mean, rstd, ops.NDBuffer.empty((0, 16)))
    assert y.shape == (0, 16) and not down(gw).any() and not down(gb).any()


# ---- attention --------------------------------------------------------------------------------------------------------------------


def attention_reference(q, k, v, scale, causal, lengths, starts, dout):
    """out, lse and gradients by autograd in 64 bits, a row at a time over the keys that it may use: nothing else is touched."""
    B, n, H, D = q.shape
    m, group = k.shape[1], H // k.shape[2]
    q, k, v = (t.double().contiguous().requires_grad_(True) for t in (q, k, v))
    out, lse = [], torch.full((B, H, n), -math.inf, dtype=torch.float64)
    for b in range(B):
        length = m if lengths is None else min(max(int(lengths[b]), 0), m)
        first = m - n if starts is None else int(starts[b])
        limit = torch.full((n,), length) if not causal else (first + torch.arange(n) + 1).clamp(0, length)
        kk, vv = (t[b, :length].repeat_interleave(group, 1).transpose(0, 1) for t in (k, v))  # [H, length, D]
        ok = torch.arange(length)[None, :] < limit[:, None]
        s = (q[b].transpose(0, 1) @ kk.transpose(1, 2) * scale).masked_fill(~ok, -math.inf)
        some = limit > 0
        z = 0.0 * q[b].transpose(0, 1)
        if bool(some.any()):
            p = torch.softmax(s[:, some], -1)
            z = z.index_put((torch.arange(H)[:, None], torch.nonzero(some)[:, 0][None, :]), p @ vv)
            lse[b][:, some] = torch.logsumexp(s[:, some].detach(), -1)
        out.append(z.transpose(0, 1))
    out = torch.stack(out)
    if dout is not None:
        out.backward(dout.double())
    zero = lambda t: t.grad if t.grad is not None else torch.zeros_like(t)  # noqa: E731
    return out.detach().numpy(), lse.numpy(), [zero(t).numpy() for t in (q, k, v)]


ATTENTION = [  # batch, queries, keys, heads, kv_heads, dim, causal, lengths, starts
    (1, 1, 1, 1, 1, 1, False, None, None),
    (2, 1, 7, 3, 1, 5, False, None, None),
    (2, 5, 5, 4, 4, 8, True, None, None),
    (3, 1, 1000, 4, 2, 64, False, [1000, 1, 333], None),
    (2, 1, 5000, 8, 1, 128, False, [4999, 0], None),
    (1, 3, 2100, 6, 3, 80, True, [2000], [1997]),
    (2, 33, 33, 4, 4, 32, False, [33, 0], None),
    (2, 64, 64, 2, 2, 64, True, None, None),
    (1, 65, 127, 2, 1, 33, True, None, None),
    (2, 100, 60, 4, 2, 40, True, None, None),      # the first 40 queries have no keys
    (3, 50, 90, 2, 2, 16, True, [90, 20, 5], [40, -30, 0]),
    (1, 127, 300, 4, 4, 127, False, [257], None),
    (2, 200, 200, 2, 2, 128, True, [131, 200], [0, 0]),
    (1, 333, 333, 8, 2, 96, True, None, None),
    (1, 700, 513, 2, 1, 64, False, None, None),
    (2, 129, 257, 3, 3, 72, True, [-5, 400], [1000000, -1000000]),
    (9, 65, 65, 8, 2, 33, True, [65, 64, 0, 1, 33, 65, 50, 2, 32], None),
    (8, 160, 96, 16, 8, 64, True, None, None),     # the first 64 queries have no keys
    (6, 97, 290, 16, 16, 20, True, [290, 100, 64, 0, 289, 97], [193, 3, -33, 10, 192, 0]),
    (4, 130, 400, 16, 16, 100, False, [1, 257, 399, 128], None),
    (1, 300, 300, 24, 3, 128, True, None, None),
    (3, 384, 384, 8, 8, 64, True, [384, 255, 129], None),
    (1, 100, 9000, 8, 8, 64, True, [8190], [8090]),  # few query tiles: the keys in runs
    (8, 300, 310, 16, 8, 20, True, [310, 299, 0, 1, 64, 65, 300, 128], [10, 10, 10, -299, 0, -3, 200, 5]),
    (3, 700, 260, 12, 4, 65, True, [260, 17, 0], None),  # the first 440 queries have no keys
    (2, 260, 1500, 12, 4, 127, False, [1500, 700], None),
]


def attention_case(seed, case):
    B, n, m, H, Hk, D = case[:6]
    return randn(seed, B, n, H, D), randn(seed + 1, B, m, Hk, D), randn(seed + 2, B, m, Hk, D), randn(seed + 3, B, n, H, D)


def ints(values):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: "-".join(str(x) for x in c[:7]))
def test_attention(ops, case):
    causal, lengths, starts = case[6:]
    q, k, v, dout = attention_case(11, case)
    scale = 1.3 / math.sqrt(case[5])
    want, want_lse, grads = attention_reference(q, k, v, scale, causal, lengths, starts, dout)
    Q, K, V, DO = (up(ops, t) for t in (q, k, v, dout))
    mask = dict(scale=scale, causal=causal, key_lengths=ints(lengths), query_starts=ints(starts))
    o, lse = ops.A.attention(Q, K, V, **mask)
    close(down(o), want, RTOL_FRO, "out")
    close(down(lse), want_lse, RTOL_FRO, "lse")
    got = ops.A.attention_backward(Q, K, V, o, lse, DO, **mask)
    for g, ref, what in zip(got, grads, ("grad_q", "grad_k", "grad_v")):
        if case[2] > 1 or what == "grad_v":  # a lone key has probability one: its gradients to q and k are zero but for rounding
            close(down(g), ref, 2 * RTOL_FRO, what)
    only, none = ops.A.attention(Q, K, V, statistics=False, **mask)
    assert none is None and torch.equal(down(only), down(o))
    again = ops.A.attention_backward(Q, K, V, o, lse, DO, **mask)
    assert all(torch.equal(down(a), down(b)) for a, b in zip(got, again))
    for skip in range(3):  # one gradient at a time gives the same bits
        some = ops.A.attention_backward(Q, K, V, o, lse, DO, need=[i == skip for i in range(3)], **mask)
        assert [s is not None for s in some] == [i == skip for i in range(3)] and torch.equal(down(some[skip]), down(got[skip]))


@pytest.mark.parametrize("case", [
    (1, 2100, 130, 2, 1, 20, False, None, None),    # the queries of a block of keys in runs
    (2, 1111, 257, 3, 3, 64, True, [257, 100], [-200, -1000]),
    (1, 150, 3001, 2, 2, 40, True, [2900], [2000]),  # the keys of a block of queries in runs
    (1, 1025, 1300, 4, 2, 128, True, None, None),   # both
    (2, 900, 900, 2, 1, 96, True, [900, 0], None),
], ids=lambda c: "-".join(str(x) for x in c[:7]))
@pytest.mark.parametrize("bad", [None, "k", "q"])
def test_attention_gradients_in_runs(ops, case, bad):
    """Few heads: the parts of the runs add up, also into what is there, one gradient at a time, and for heads that are computed value by value (a value far out, of which p is nearly zero)."""
    causal, lengths, starts = case[6:]
    q, k, v, dout = attention_case(17, case)
    if bad == "k":
        k[0, 77, 0, 3] = 1.0e9
        q[0, :, :case[3] // case[4], 3] = -q[0, :, :case[3] // case[4], 3].abs() - 0.01  # (so that the key has no weight)
    elif bad == "q":
        dout[0, 33, 0, 0] = 3.0e8
    scale = 1.1 / math.sqrt(case[5])
    want, _, grads = attention_reference(q, k, v, scale, causal, lengths, starts, dout)
    Q, K, V, DO = (up(ops, t) for t in (q, k, v, dout))
    mask = dict(scale=scale, causal=causal, key_lengths=ints(lengths), query_starts=ints(starts))
    o, lse = ops.A.attention(Q, K, V, **mask)
    close(down(o), want, RTOL_FRO, "out")
    got = ops.A.attention_backward(Q, K, V, o, lse, DO, **mask)
    base = [randn(40 + i, *t.shape) for i, t in enumerate((q, k, v))]
    for skip, (g, ref, what) in enumerate(zip(got, grads, ("grad_q", "grad_k", "grad_v"))):
        close(down(g), ref, 2 * RTOL_FRO, what)
        some = ops.A.attention_backward(Q, K, V, o, lse, DO, need=[i == skip for i in range(3)], **mask)
        assert torch.equal(down(some[skip]), down(g))
    into = [up(ops, t) for t in base]
    ops.A.attention_backward(Q, K, V, o, lse, DO, into=into, **mask)
    for g, i, t in zip(got, into, base):
        assert torch.equal(down(i), down(g) + t)


def test_attention_gradients_of_long_sums(ops):
    """Runs of 128 tiles at the most: the sums over a run round six times a tile, by half a step of the sum so far, which grows as a random walk does: sqrt(6 * 128 / 2) 2^-24 of the result."""
    B, n, m, H, Hk, D = 1, 8192, 4000, 8, 2, 32
    q, k, v, dout = (t.cuda() for t in attention_case(23, (B, n, m, H, Hk, D)))
    Q, K, V, DO = (up(ops, t) for t in (q, k, v, dout))
    o, lse = ops.A.attention(Q, K, V, scale=0.1)
    got = [down(t) for t in ops.A.attention_backward(Q, K, V, o, lse, DO, scale=0.1)]
    q, k, v, dout = (t.double().transpose(1, 2)[0].contiguous() for t in (q, k, v, dout))  # [heads, rows, D]
    want = [torch.zeros_like(t) for t in (q, k, v)]
    for h in range(H):
        kk, vv = k[h * Hk // H], v[h * Hk // H]
        p = torch.softmax(0.1 * (q[h] @ kk.t()), -1)
        want[2][h * Hk // H] += p.t() @ dout[h]
        ds = p * (dout[h] @ vv.t())
        ds -= p * ds.sum(-1, keepdim=True)
        want[0][h] = 0.1 * (ds @ kk)
        want[1][h * Hk // H] += 0.1 * (ds.t() @ q[h])
    for g, ref, what in zip(got, want, ("grad_q", "grad_k", "grad_v")):
        close(g, ref.transpose(0, 1)[None].cpu().numpy(), math.sqrt(6 * 128 / 2) * 2.0 ** -24, what)


@pytest.mark.parametrize("n", [1, 40, 150, 600])
def test_attention_of_strided_operands(ops, n):
    """Slices of a joint projection, heads before positions, every second value of d, a batch that is one sequence repeated (stride 0)."""
    B, H, Hk, D, m = 2, 4, 2, 24, max(150, n)
    qkv = randn(3, B, m, (H + 2 * Hk) * D)
    packed = (qkv[:, m - n:, :H * D].unflatten(2, (H, D)), qkv[:, :, H * D:(H + Hk) * D].unflatten(2, (Hk, D)), qkv[:, :, (H + Hk) * D:].unflatten(2, (Hk, D)))
    swapped = tuple(randn(4 + i, B, h, s, D).transpose(1, 2) for i, (h, s) in enumerate(((H, n), (Hk, m), (Hk, m))))
    every = tuple(randn(8 + i, B, s, h, 2 * D)[..., ::2] for i, (h, s) in enumerate(((H, n), (Hk, m), (Hk, m))))
    shared = (randn(14, B, n, H, D), randn(12, 1, m, Hk, D).expand(B, -1, -1, -1), randn(13, 1, m, Hk, D).expand(B, -1, -1, -1))
    dout = randn(20, B, n, H, D)
    for q, k, v in (packed, swapped, every, shared):
        want, want_lse, grads = attention_reference(q, k, v, 0.2, True, None, None, dout)
        Q, K, V, DO = (up(ops, t) for t in (q, k, v, dout))
        o, lse = ops.A.attention(Q, K, V, scale=0.2, causal=True)
        close(down(o), want, RTOL_FRO, "out")
        close(down(lse), want_lse, RTOL_FRO, "lse")
        # gradients into strided places, added to what is there, nothing beside them touched
        bases = [randn(30 + i, *b.shape[:3], b.shape[3] + 3) for i, b in enumerate((q, k, v))]
        into = [up(ops, b[..., 1:-2]) for b in bases]
        ops.A.attention_backward(Q, K, V, o, lse, DO, scale=0.2, causal=True, into=into)
        for g, base, ref, what in zip(into, bases, grads, ("grad_q", "grad_k", "grad_v")):
            whole = g.storage.cpu().reshape(base.shape)
            assert torch.equal(whole[..., :1], base[..., :1]) and torch.equal(whole[..., -2:], base[..., -2:])
            # (two roundings of the sum beside the gradient's own error)
            close(whole[..., 1:-2] - base[..., 1:-2].double(), ref, 2 * RTOL_FRO + 2.0 ** -23 * np.linalg.norm(base[..., 1:-2]) / np.linalg.norm(ref), what)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 3.0e38])
@pytest.mark.parametrize("n", [1, 70, 100])
def test_keys_that_are_not_allowed_are_not_used(ops, bad, n):
    """Whatever lies behind a sequence's keys, or ahead of a query, leaves no trace."""
    B, m, H, D = 2, 140, 2 if n < 100 else 64, 64
    q, k, v, dout = randn(1, B, n, H, D), randn(2, B, m, H, D), randn(3, B, m, H, D), randn(4, B, n, H, D)
    lengths, starts = [100, 37], [100 - n, 20 - n]
    want = attention_reference(q, k, v, 0.1, True, lengths, starts, dout)
    for t in (k, v):
        t[0, 100:] = bad
        t[1, 20:] = bad  # the last query of the second sequence is at position 19
    Q, K, V, DO = (up(ops, t) for t in (q, k, v, dout))
    mask = dict(scale=0.1, causal=True, key_lengths=ints(lengths), query_starts=ints(starts))
    o, lse = ops.A.attention(Q, K, V, **mask)
    close(down(o), want[0], RTOL_FRO, "out")
    close(down(lse), want[1], RTOL_FRO, "lse")
    for g, ref, what in zip(ops.A.attention_backward(Q, K, V, o, lse, DO, **mask), want[2], ("grad_q", "grad_k", "grad_v")):
        close(down(g), ref, 2 * RTOL_FRO, what)


@pytest.mark.parametrize("bad", [math.nan, math.inf, 1.0e30, 1.0e9])
@pytest.mark.parametrize("where", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("dim", [16, 64, 96, 128])
def test_a_row_out_of_the_ordinary_stays_with_what_sees_it(ops, where, bad, dim):
    """One row of one head that is not finite, or far larger than all others: queries before it, keys behind it and the other heads are as without it."""
    B, n, H, at = 2, 200, 24 if dim > 32 else 48, 120  # enough for the kernels in tiles
    tensors = {name: randn(i, B, n, H, dim) for i, name in enumerate(("q", "k", "v", "dout"))}
    want = attention_reference(tensors["q"], tensors["k"], tensors["v"], 0.2, True, None, None, tensors["dout"])
    tensors[where][1, at, 0] = bad
    Q, K, V, DO = (up(ops, tensors[name]) for name in ("q", "k", "v", "dout"))
    o, lse = ops.A.attention(Q, K, V, scale=0.2, causal=True)
    grads = ops.A.attention_backward(Q, K, V, o, lse, DO, scale=0.2, causal=True)
    key = where in ("k", "v")
    for got, ref, by_query, what in ((o, want[0], True, "out"), (grads[0], want[2][0], True, "grad_q"), (grads[1], want[2][1], False, "grad_k"), (grads[2], want[2][2], False, "grad_v")):
        clean = np.ones((B, n, H), bool)
        if by_query:
            clean[1, at:, 0] = not key  # a key's row is seen by the queries from it on, a query's by itself
            clean[1, at, 0] = False
        else:
            clean[1, :, 0] = False  # every key is seen by such a query, or shares the queries from it on
            clean[1, at + 1:, 0] = not key
        close(np.asarray(down(got))[clean], ref[clean], RTOL_FRO if what == "out" else 2 * RTOL_FRO, what)


def test_attention_with_values_that_are_not_finite(ops):
    """An allowed key that is not a number reaches the queries that see it, and no other sequence or head."""
    B, n, H, D = 2, 80, 2, 32
    q, k, v = randn(1, B, n, H, D), randn(2, B, n, H, D), randn(3, B, n, H, D)
    want = attention_reference(q, k, v, 0.2, True, None, None, None)[0]
    k[1, 50, 0, 3] = math.nan
    o, lse = (down(t).numpy() for t in ops.A.attention(up(ops, q), up(ops, k), up(ops, v), scale=0.2, causal=True))
    assert np.isnan(o[1, 50:, 0]).all() and np.isnan(lse[1, 0, 50:]).all()
    o[1, 50:, 0] = want[1, 50:, 0]
    close(o, want, RTOL_FRO, "the others")


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30, 2.0 ** -120])
@pytest.mark.parametrize("n", [3, 160])
def test_attention_scales(ops, n, scale):
    """No scale (every allowed key counts the same), a negative one, and ones that no score survives."""
    q, k, v, dout = (randn(i, 1, n, 2, 64) for i in range(4))
    want, want_lse, grads = attention_reference(q, k, v, scale, True, None, None, dout)
    for reps in (1, 40):  # enough heads for either kernel
        Qr, Kr, Vr, DOr = (up(ops, t.repeat(reps, 1, 1, 1)) for t in (q, k, v, dout))
        o, lse = ops.A.attention(Qr, Kr, Vr, scale=scale, causal=True)
        close(down(o)[-1], want[0], RTOL_FRO, "out")
        close(down(lse)[-1], want_lse[0], RTOL_FRO, "lse")
        got = ops.A.attention_backward(Qr, Kr, Vr, o, lse, DOr, scale=scale, causal=True)
        for g, ref, what in zip(got, grads, ("grad_q", "grad_k", "grad_v")):
            if what == "grad_v" or abs(scale) > 1e-20:
                close(down(g)[-1], ref[0], 2 * RTOL_FRO, what)
            else:
                assert np.abs(down(g)[-1].numpy()).max() <= abs(scale) * 1e4


@pytest.mark.parametrize("size", [2.0 ** -108, 2.0 ** 90])
@pytest.mark.parametrize("reps", [1, 60])
def test_attention_gradients_of_any_size(ops, reps, size):
    """Upstream gradients far from one: the gradients are those of one times as much."""
    q, k, v, dout = (randn(i, 1, 160, 2, 64) for i in range(4))
    want = attention_reference(q, k, v, 0.11, True, None, None, dout)[2]
    Q, K, V, DO = (up(ops, t.repeat(reps, 1, 1, 1)) for t in (q, k, v, dout * size))
    o, lse = ops.A.attention(Q, K, V, scale=0.11, causal=True)
    for g, ref, what in zip(ops.A.attention_backward(Q, K, V, o, lse, DO, scale=0.11, causal=True), want, ("grad_q", "grad_k", "grad_v")):
        close(down(g)[-1].double() / size, ref[0], 2 * RTOL_FRO, what)


def test_attention_extreme_scores(ops):
    """Scores of thousands and values over 40 powers of two: the maximum is taken off before the exponential, and the sums have fp32's range."""
    B, n, H, D = 1, 96, 2, 64
    q, k, v, dout = randn(1, B, n, H, D) * 16, randn(2, B, n, H, D) * 16, randn(3, B, n, H, D), randn(4, B, n, H, D)
    v[:, :, 1] *= 2.0 ** 40
    dout[:, :, 0] *= 2.0 ** -40
    want = attention_reference(q, k, v, 1.0, True, None, None, dout)
    # The magnitudes of a score's 64 products add up to 64 * 16 * 16 * 0.64 * 2 = 21000 at most; 12 roundings of 2^-24 of that are 2^-6, in the exponent and so
    # relative in p.  Nearly every p is 0 or 1, and a gradient p (dP - delta) cancels where it is 1: its error is measured against p (|dP| + |delta|).
    tol = 2.0 ** -6
    for reps in (1, 150):  # enough heads for either kernel
        Q, K, V, DO = (up(ops, t.repeat(reps, 1, 1, 1)) for t in (q, k, v, dout))
        o, lse = ops.A.attention(Q, K, V, scale=1.0, causal=True)
        close(down(lse)[-1], want[1][0], RTOL_FRO, "lse")
        got = [down(g)[-1] for g in ops.A.attention_backward(Q, K, V, o, lse, DO, scale=1.0, causal=True)]
        for h in range(H):
            close(down(o)[-1, :, h], want[0][0, :, h], tol, "out")
            close(got[2][:, h], want[2][2][0, :, h], tol, "grad_v")
            qh, kh, vh, gh = (t[0, :, h].double().numpy() for t in (q, k, v, dout))
            p = np.tril(np.exp(np.minimum(qh @ kh.T - want[1][0, h][:, None], 0.0)))
            terms = p * (np.abs(gh @ vh.T) + np.abs((gh * want[0][0, :, h]).sum(1))[:, None])
            for g, ref, size, what in ((got[0], want[2][0], terms @ np.abs(kh), "grad_q"), (got[1], want[2][1], terms.T @ np.abs(qh), "grad_k")):
                assert np.linalg.norm(g[:, h].numpy() - ref[0, :, h]) <= tol * np.linalg.norm(size), what


@pytest.mark.parametrize("size", [1.0, 2.0 ** -112])
@pytest.mark.parametrize("H", [2, 40])
def test_attention_blocks_of_keys_of_different_sizes(ops, H, size):
    """Keys and values whose blocks of 64 lie up to 2^15 apart, one of zeros among them, each query with its weight in one block: every row of the result is right against its own size."""
    B, n, m, D = 1, 300, 256, 64
    q, k, v = randn(1, B, n, H, D), randn(2, B, m, H, D) * 0.2, randn(3, B, m, H, D)
    q[..., :4] = k[..., :4] = 0.0
    for b, factor in enumerate((2.0 ** -6, 2.0 ** 7, 2.0 ** -8, 1.0)):
        v[:, 64 * b:64 * b + 64] *= size * factor
        q[:, b::4, :, b] = 32.0 * 2.0 ** (b % 3 * 4)
        k[:, 64 * b:64 * b + 64, :, b] = 2.0 ** -(b % 3 * 4)
    k, v = (torch.cat((t[:, :128], 0.0 * t[:, :64], t[:, 128:]), 1) for t in (k, v))  # the zeros' scores are 0, the others' of a query 32 and near 0
    want, want_lse, _ = attention_reference(q, k, v, 1.0, False, None, None, None)
    o, lse = ops.A.attention(up(ops, q), up(ops, k), up(ops, v), scale=1.0)
    close(down(lse), want_lse, RTOL_FRO, "lse")
    # (a score of 32, made of products that cancel to a part in ten at the most, is right to 12 roundings of 2^-24 of 40, and so is its weight)
    error = np.linalg.norm(down(o).numpy() - want, axis=-1) / np.linalg.norm(want, axis=-1)
    assert error.max() <= 12 * 40 * 2.0 ** -24, error.max()


def test_attention_without_keys_or_queries(ops):
    q, none = up(ops, randn(1, 2, 3, 2, 8)), ops.NDBuffer.empty((2, 0, 2, 8))
    o, lse = ops.A.attention(q, none, none)
    assert not down(o).any() and torch.isneginf(down(lse)).all()
    gq, gk, gv = ops.A.attention_backward(q, none, none, o, lse, q)
    assert not down(gq).any() and gk.shape == (2, 0, 2, 8)
    k, empty = up(ops, randn(2, 2, 5, 2, 8)), ops.NDBuffer.empty((2, 0, 2, 8))
    o, lse = ops.A.attention(empty, k, k)
    assert o.shape == (2, 0, 2, 8) and lse.shape == (2, 2, 0)
    gq, gk, gv = ops.A.attention_backward(empty, k, k, o, lse, empty)
    assert not down(gk).any() and not down(gv).any()


@pytest.mark.parametrize("n", [1, 130, 2300, 5000])
def test_attention_offsets_past_32_bits(ops, n):
    """A cache whose positions lie 2^24 values apart: the last of 300 is more than 2^32 values behind the first."""
    m, D, pitch = 300, 64, 1 << 24
    k, v, q = randn(1, 1, m, 1, D), randn(2, 1, m, 1, D), randn(3, 1, n, 1, D)
    store = torch.empty(m * pitch + 2 * D, dtype=torch.float32, device="cuda")
    places = [store.as_strided((1, m, 1, D), (0, pitch, D, 1), off) for off in (0, D)]
    places[0].copy_(k)
    places[1].copy_(v)
    K, V = (ops.NDBuffer(store, (1, m, 1, D), (0, pitch, D, 1), off) for off in (0, D))
    o, lse = ops.A.attention(up(ops, q), K, V, scale=0.125, causal=True)
    dout = randn(4, 1, n, 1, D)
    want = attention_reference(q, k, v, 0.125, True, None, None, dout)
    close(down(o), want[0], RTOL_FRO, "out")
    for g, ref, what in zip(ops.A.attention_backward(up(ops, q), K, V, o, lse, up(ops, dout), scale=0.125, causal=True), want[2], ("grad_q", "grad_k", "grad_v")):
        close(down(g), ref, 2 * RTOL_FRO, what)


# ---- vocabulary loss -----------------------------------------------------------------------------------------------------------------


def vocabulary_reference(h, w, b, target, ignore, smoothing, reduction, upstream):
    h, w, b = (None if t is None else t.double().contiguous().requires_grad_(True) for t in (h, w, b))
    x = h @ w
    x = x + b if b is not None else x
    lse = torch.logsumexp(x, -1)
    valid = target != ignore
    t = torch.where(valid, target, 0).long()
    loss = (1 - smoothing) * (lse - x.gather(1, t[:, None])[:, 0]) + (smoothing * (lse - x.mean(-1)) if smoothing else 0.0)
    loss = torch.where(valid, loss, 0.0)
    total = {"none": loss, "sum": loss.sum(), "mean": loss.sum() / max(1, int(valid.sum()))}[reduction]
    (total * upstream.double().reshape(total.shape)).sum().backward()
    return loss.detach().numpy(), lse.detach().numpy(), int(valid.sum()), [None if p is None else p.grad.numpy() for p in (h, w, b)]


VOCABULARY = [  # tokens, dim, vocabulary, weight, bias, reduction, smoothing, int64 targets
    (1, 1, 1, "dense", False, "sum", 0.0, True),
    (1, 7, 3, "dense", True, "mean", 0.1, False),
    (5, 16, 17, "tied", True, "none", 0.0, True),
    (64, 128, 1000, "tied", False, "mean", 0.0, True),
    (2, 50, 4099, "tied", True, "mean", 0.1, True),
    (31, 257, 129, "strided", True, "sum", 0.0, True),
    (32, 96, 1281, "dense", True, "none", 0.1, False),
    (33, 31, 640, "tied", True, "mean", 0.0, True),
    (63, 130, 1025, "dense", True, "sum", 0.3, True),
    (65, 64, 1000, "tied", True, "mean", 0.1, True),
    (128, 64, 256, "dense", True, "mean", 0.0, False),
    (129, 100, 257, "dense", True, "sum", 0.1, True),
    (255, 33, 511, "tied", True, "none", 0.2, False),
    (300, 130, 2049, "strided", True, "mean", 0.1, True),
    (77, 769, 1500, "tied", True, "mean", 1.0, True),
    (513, 48, 5003, "dense", False, "none", 0.0, True),
    (1900, 65, 12001, "tied", True, "mean", 0.1, False),
    (2500, 100, 8003, "dense", True, "sum", 0.1, True),
    (4100, 33, 9000, "strided", True, "none", 0.0, True),
    (2000, 769, 1501, "tied", False, "mean", 1.0, True),
    (3000, 40, 130, "tied", True, "none", 0.1, True),     # few tiles of the weight's gradient: the tokens in runs
    (3001, 150, 300, "strided", False, "mean", 0.0, True),
    (1500, 130, 1500, "dense", True, "mean", 0.0, True),  # forward and backward by different kernels
]


def vocabulary_case(case, seed=5):
    m, d, v, weight = case[:4]
    h = randn(seed, m, d)
    scale = 1.5 / math.sqrt(d)
    w = {"dense": lambda: randn(seed + 1, d, v) * scale, "tied": lambda: (randn(seed + 1, v, d) * scale).t(), "strided": lambda: (randn(seed + 1, d, 2 * v) * scale)[:, ::2]}[weight]()
    g = torch.Generator().manual_seed(seed)
    target = torch.randint(0, v, (m,), generator=g)
    target[torch.rand(m, generator=g) < 0.1] = -100
    upstream = randn(seed + 3, m) if case[5] == "none" else torch.tensor([0.7])
    return h, w, (randn(seed + 2, v) if case[4] else None), target if case[7] else target.int(), upstream


@pytest.mark.parametrize("case", VOCABULARY, ids=lambda c: "-".join(str(x) for x in c))
def test_vocabulary_loss(ops, case):
    m, d, v, weight, _, reduction, smoothing, _ = case
    h, w, b, target, upstream = vocabulary_case(case)
    loss, lse, count, grads = vocabulary_reference(h, w, b, target, -100, smoothing, reduction, upstream)
    H, W, B, T, U = up(ops, h), up(ops, w), up(ops, b), target.cuda(), upstream.cuda()
    assert (W.strides[0] == 1) == (weight == "tied" or v == 1)
    got = ops.V.vocabulary_loss(H, W, B, T, label_smoothing=smoothing)
    # a loss is the difference of two logits' size of numbers: measured against those
    assert np.abs(down(got.per_sample).numpy() - loss).max() <= 2 * RTOL_FRO * max(1.0, np.abs(lse).max())
    assert np.array_equal(down(got.per_sample).numpy()[(target == -100).numpy()], np.zeros(int((target == -100).sum()), np.float32))
    assert np.abs(down(got.lse).numpy() - lse).max() <= RTOL_FRO * max(1.0, np.abs(lse).max())
    assert int(got.valid_count.item()) == count and abs(float(down(got.loss_sum)[0]) - loss.sum()) <= 2 * RTOL_FRO * max(1.0, np.abs(lse).max()) * m
    back = ops.V.vocabulary_loss_backward(H, W, B, T, got, U, reduction=reduction, label_smoothing=smoothing)
    for g, ref, what in zip(back, grads, ("grad_h", "grad_w", "grad_bias")):
        assert (g is None) == (ref is None)
        # one word: its probability is one and the gradient zero but for rounding
        if g is not None and v > 1:
            close(down(g), ref, 2 * RTOL_FRO, what)
    again = ops.V.vocabulary_loss_backward(H, W, B, T, got, U, reduction=reduction, label_smoothing=smoothing)
    assert all(a is None or torch.equal(down(a), down(g)) for a, g in zip(again, back))
    # added to what is there; a weight gradient with strides of its own
    olds = [randn(40, m, d), randn(41, d, 2 * v + 1)[:, 1::2], randn(42, v)]
    into = [up(ops, olds[0]), up(ops, olds[1]), up(ops, olds[2]) if b is not None else None]
    ops.V.vocabulary_loss_backward(H, W, B, T, got, U, reduction=reduction, label_smoothing=smoothing, into=into)
    for g, one, old in zip(into, back, olds):
        if g is not None:
            close(down(g), down(one).double().numpy() + old.double().numpy(), 2.0 ** -23, "accumulated")


def test_vocabulary_loss_in_several_pieces(ops, monkeypatch):
    """Tokens enough for more than one piece of the vocabulary: 2^28 values of G are 20480 tokens times 13107 words."""
    m, d, v = 20480, 32, 14001
    h, w, b = randn(1, m, d).cuda(), (randn(2, v, d) * 0.3).cuda(), randn(3, v).cuda()
    target = torch.randint(0, v, (m,), generator=torch.Generator().manual_seed(1)).cuda()
    x = h.double() @ w.double().t() + b.double()
    lse = torch.logsumexp(x, -1)
    g = torch.exp(x - lse[:, None])
    g[torch.arange(m), target] -= 1.0
    g /= m
    H, W, B = ops.NDBuffer(h.view(-1), (m, d)), ops.NDBuffer(w.view(-1), (v, d)).transpose(), ops.NDBuffer(b, (v,))
    got = ops.V.vocabulary_loss(H, W, B, target)
    one = torch.ones(1, device="cuda")
    for weight in (W, ops.NDBuffer(w.t().contiguous().view(-1), (d, v))):
        gh, gw, gb = ops.V.vocabulary_loss_backward(H, weight, B, target, got, one)
        close(down(got.lse), lse.cpu().numpy(), RTOL_FRO, "lse")
        close(down(gh), (g @ w.double()).cpu().numpy(), 2 * RTOL_FRO, "grad_h")
        close(down(gw), (h.double().t() @ g).cpu().numpy(), 2 * RTOL_FRO, "grad_w")
        close(down(gb), g.sum(0).cpu().numpy(), 2 * RTOL_FRO, "grad_bias")


def test_vocabulary_loss_targets(ops):
    """Every target ignored; targets outside the vocabulary; an ignore_index inside it."""
    h, w = randn(1, 20, 24), randn(2, 24, 50)
    H, W, one = up(ops, h), up(ops, w), torch.ones(1, device="cuda")
    t = torch.full((20,), -100, dtype=torch.int64, device="cuda")
    loss = ops.V.vocabulary_loss(H, W, None, t)
    assert int(loss.valid_count.item()) == 0 and float(down(loss.loss_sum)[0]) == 0.0
    gh, gw, _ = ops.V.vocabulary_loss_backward(H, W, None, t, loss, one)
    assert not down(gh).any() and not down(gw).any()
    t = torch.arange(20, device="cuda")
    t[3], t[7], t[11] = 50, -1, 7
    t[12] = 7
    loss = ops.V.vocabulary_loss(H, W, None, t, ignore_index=7)
    each = down(loss.per_sample).numpy()
    assert np.isnan(each[[3, 7]]).all() and not each[[11, 12]].any() and np.isfinite(np.delete(each, [3, 7])).all() and int(loss.valid_count.item()) == 18


@pytest.mark.parametrize("m, v", [(12, 700), (50, 700), (150, 700), (2100, 9000)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, 1.0e30])
def test_vocabulary_loss_rows_that_do_not_count(ops, bad, m, v):
    """Whatever the hidden state of an ignored token holds, the others' losses and all gradients are as without it; and a row far larger than the others
    takes nothing from their losses."""
    d = 48
    h, w, b = randn(1, m, d), randn(2, v, d) * 0.2, randn(3, v)
    target = torch.arange(m)
    target[[3, m - 1]] = -100
    want = vocabulary_reference(h, w.t(), b, target, -100, 0.1, "mean", torch.ones(1))
    h[3], h[m - 1] = bad, -bad
    H, W, B, T = up(ops, h), up(ops, w).transpose(), up(ops, b), target.cuda()
    loss = ops.V.vocabulary_loss(H, W, B, T, label_smoothing=0.1)
    assert np.abs(down(loss.per_sample).numpy() - want[0]).max() <= 2 * RTOL_FRO * np.abs(want[1]).max()
    back = ops.V.vocabulary_loss_backward(H, W, B, T, loss, torch.ones(1, device="cuda"), label_smoothing=0.1)
    for g, ref, what in zip(back, want[3], ("grad_h", "grad_w", "grad_bias")):
        close(down(g), ref, 2 * RTOL_FRO, what)
    if math.isfinite(bad):
        target[3] = 5
        loss = ops.V.vocabulary_loss(H, W, B, target.cuda(), label_smoothing=0.1)
        keep = np.arange(m) != 3
        assert np.abs(down(loss.per_sample).numpy() - want[0])[keep].max() <= 2 * RTOL_FRO * np.abs(want[1]).max()


@pytest.mark.parametrize("m, v", [(20, 700), (40, 700), (100, 700), (2300, 12000)])
def test_vocabulary_loss_words_shut_out_by_the_bias(ops, m, v):
    """A bias of -inf gives a word no probability, and of its type's lowest value next to none; all but one: the loss of that one is zero."""
    d = 32
    h, w, b = randn(1, m, d), randn(2, d, v), randn(3, v)
    b[600:] = -math.inf
    b[300:400] = torch.finfo(torch.float32).min
    target = torch.arange(m) % 300
    want = vocabulary_reference(h, w, b, target, -100, 0.0, "sum", torch.ones(1))
    H, W, B, T, one = up(ops, h), up(ops, w), up(ops, b), target.cuda(), torch.ones(1, device="cuda")
    loss = ops.V.vocabulary_loss(H, W, B, T)
    close(down(loss.lse), want[1], RTOL_FRO, "lse")
    for g, ref, what in zip(ops.V.vocabulary_loss_backward(H, W, B, T, loss, one, reduction="sum"), want[3], ("grad_h", "grad_w", "grad_bias")):
        close(down(g), ref, 2 * RTOL_FRO, what)
    b[1:] = -math.inf
    loss = ops.V.vocabulary_loss(H, W, up(ops, b), torch.zeros(m, dtype=torch.int64, device="cuda"))
    assert np.abs(down(loss.per_sample).numpy()).max() <= RTOL_FRO * 10


@pytest.mark.parametrize("m, v", [(50, 600), (100, 600), (1700, 9000)])
@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -30, 2.0 ** 60])
def test_vocabulary_loss_scales(ops, scale, m, v):
    """Hidden states and weights far from one whose products are ordinary: the halves are scaled by the largest value."""
    d = 64
    h, w, target = randn(1, m, d) * scale, randn(2, d, v) * 0.2 / scale, torch.arange(m)
    want = vocabulary_reference(h, w, None, target, -100, 0.0, "sum", torch.ones(1))
    H, W, T, one = up(ops, h), up(ops, w), target.cuda(), torch.ones(1, device="cuda")
    loss = ops.V.vocabulary_loss(H, W, None, T)
    close(down(loss.lse), want[1], RTOL_FRO, "lse")
    for g, ref, what in zip(ops.V.vocabulary_loss_backward(H, W, None, T, loss, one, reduction="sum"), want[3], ("grad_h", "grad_w")):
        close(down(g), ref, 2 * RTOL_FRO, what)


# ---- together, streams, graphs --------------------------------------------------------------------------------------------------------


def block_tensors(ops, B=2, S=37, E=48, H=4, V=211, seed=1):
    from tenmo_amd.net import Linear

    rng = np.random.default_rng(seed)
    h = ops.Tensor.from_numpy(rng.standard_normal((B, S, E), dtype=np.float32), requires_grad=True)
    norm, qkv, head_norm = ops.N.LayerNorm(E), Linear(E, 3 * E, rng), ops.N.LayerNorm(E)
    emb = ops.Tensor.from_numpy(0.3 * rng.standard_normal((V, E), dtype=np.float32), requires_grad=True)
    for p in norm.parameters() + head_norm.parameters():
        p.buffer.storage += 0.1 * torch.from_numpy(rng.standard_normal(E, dtype=np.float32)).cuda()
    target = torch.from_numpy(rng.integers(0, V, B * S)).cuda()
    return h, norm, qkv, head_norm, emb, target, H


def test_a_training_step_of_them(ops):
    """norm -> joint projection -> causal attention -> norm -> loss over a tied vocabulary, forward and backward through the autograd graph, against
    64-bit autograd and against differences of the loss."""
    h, norm, qkv, head_norm, emb, target, H = block_tensors(ops)
    B, S, E = h.shape()

    def reference():
        leaves = [torch.from_numpy(t.to_numpy()).double().requires_grad_(True) for t in (h, norm.weight, norm.bias, qkv.weight, qkv.bias, head_norm.weight, head_norm.bias, emb)]
        x, nw, nb, w, b, hw, hb, e = leaves
        y = torch.nn.functional.layer_norm(x, (E,), nw, nb, 1e-5) @ w + b
        q, k, v = y.reshape(B, S, 3, H, E // H).permute(2, 0, 3, 1, 4)
        s = (q @ k.transpose(2, 3) / math.sqrt(E // H)).masked_fill(torch.ones(S, S).triu(1).bool(), -math.inf)
        o = (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B * S, E)
        o = torch.nn.functional.layer_norm(o, (E,), hw, hb, 1e-5)
        return torch.nn.functional.cross_entropy(o @ e.t(), target.cpu()), leaves

    def step():
        y = qkv(norm(h))
        o = ops.A.Attention.packed(y, H, causal=True)
        o = head_norm(o)
        flat = ops.Tensor(ops.NDBuffer(o.buffer.storage, (B * S, E)), requires_grad=True)
        weight = emb.transpose()
        loss = ops.V.VocabularyLoss.forward(flat, weight, None, target)
        loss.backward()
        o.backward(ops.Tensor(ops.NDBuffer(flat.gradbox.storage, (B, S, E))))
        return loss, weight

    want, leaves = reference()
    want.backward()
    loss, weight = step()
    assert abs(float(loss.to_numpy()[0]) - float(want.detach())) <= RTOL_FRO * float(want.detach())
    got = [h, norm.weight, norm.bias, qkv.weight, qkv.bias, head_norm.weight, head_norm.bias]
    # four operators in a row, each with a gradient's tolerance of its own
    for t, ref, what in zip(got, leaves, ("h", "norm.weight", "norm.bias", "qkv.weight", "qkv.bias", "head_norm.weight", "head_norm.bias")):
        close(t.grad(), ref.grad.numpy(), 8 * RTOL_FRO, what)
    close(weight.grad().T, leaves[-1].grad.numpy(), 8 * RTOL_FRO, "embedding")
    # a second backward adds
    first = h.grad().astype(np.float64)
    step()
    close(h.grad(), 2 * first, 1e-6, "twice")
    # the gradient along a direction against central differences of the loss: steps of 2^-6 leave a relative error of 2^-12 times a third derivative of the
    # size of the first, and the loss's own error of 1e-6 over a step of 2^-5 one of 3e-5
    direction = np.random.default_rng(9).standard_normal((B, S, E)).astype(np.float32)
    slope = float((first * direction).sum())
    ends = []
    for sign in (1, -1):
        h.buffer.storage += torch.from_numpy(sign * 2.0 ** -6 * direction).cuda().reshape(-1)
        ends.append(float(step()[0].to_numpy()[0]))
        h.buffer.storage -= torch.from_numpy(sign * 2.0 ** -6 * direction).cuda().reshape(-1)
    assert abs((ends[0] - ends[1]) * 2.0 ** 5 - slope) <= 0.02 * abs(slope) + 1e-4


def call_all(ops, s):
    """Every operator once, forward and backward; the buffers it returns."""
    y, mean, rstd = ops.N.layer_norm(s["x"], s["w"], s["w"])
    out = [y, mean, rstd, *ops.N.layer_norm_backward(s["x"], s["w"], mean, rstd, s["x"])]
    for q in (s["q"], s["q1"]):
        o, lse = ops.A.attention(q, s["k"], s["v"], causal=True)
        out += [o, lse, *ops.A.attention_backward(q, s["k"], s["v"], o, lse, q, causal=True)]
    loss = ops.V.vocabulary_loss(s["h"], s["e"].transpose(), s["b"], s["t"])
    out += [loss.per_sample, loss.lse, loss.loss_sum, *ops.V.vocabulary_loss_backward(s["h"], s["e"].transpose(), s["b"], s["t"], loss, s["one"])]
    few = ops.NDBuffer(s["h"].storage, (40, 80))
    loss = ops.V.vocabulary_loss(few, s["e"].transpose(), s["b"], s["t"][:40])
    out += [loss.per_sample, loss.lse, loss.loss_sum, *ops.V.vocabulary_loss_backward(few, s["e"].transpose(), s["b"], s["t"][:40], loss, s["one"])]
    return out


def state_of(ops, seed):
    s = {n: up(ops, randn(seed + i, *shape)) for i, (n, shape) in enumerate((("x", (70, 96)), ("w", (96,)), ("q", (2, 400, 8, 64)), ("k", (2, 400, 2, 64)), ("v", (2, 400, 2, 64)),
                                                                             ("q1", (2, 1, 8, 64)), ("h", (1700, 80)), ("e", (9000, 80)), ("b", (9000,))))}
    s["t"] = torch.randint(0, 9000, (1700,), generator=torch.Generator().manual_seed(seed)).cuda()
    s["one"] = torch.ones(1, device="cuda")
    return s


def bits(buffers):
    return [down(b).clone() for b in buffers]


def test_another_stream(ops):
    """Under a torch stream of one's own: inputs written there just before, results read there just behind."""
    s, t = state_of(ops, 1), state_of(ops, 2)
    want = bits(call_all(ops, t))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(3):
            for n in s:
                b = s[n] if n in ("t", "one") else s[n].storage
                torch.cuda._sleep(200000)
                b.copy_(t[n] if n in ("t", "one") else t[n].storage)
            got = [b.storage.clone() for b in call_all(ops, s)]
            for n in s:
                (s[n] if n in ("t", "one") else s[n].storage).zero_()
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a.cpu()[:b.numel()].reshape(b.shape) if b.is_contiguous() else a.cpu().as_strided(b.shape, b.stride()), b)


def test_captured_graphs(ops):
    """Two graphs with workspaces of their own, replayed in turn between eager calls on other inputs."""
    a, b = state_of(ops, 1), state_of(ops, 2)
    call_all(ops, a)
    want = [bits(call_all(ops, s)) for s in (a, b)]
    torch.cuda.synchronize()
    graphs = []
    for s in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call_all(ops, s)
        graphs.append((g, out))
    for turn in range(4):
        for (g, out), ref in zip(graphs, want):
            for o in out:
                o.storage.fill_(7.0)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(bits(out), ref)), turn
        call_all(ops, state_of(ops, 10 + turn))
        torch.cuda.synchronize()
    # new inputs in the same places
    for n in a:
        (a[n] if n in ("t", "one") else a[n].storage).copy_(b[n] if n in ("t", "one") else b[n].storage)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(bits(graphs[0][1]), want[1]))


def test_a_captured_attention_whose_sums_run_in_parts(ops):
    """Few heads, many rows: workspaces with the parts of each run, of two graphs replayed in turn and of eager calls between them."""
    def call(s):
        o, lse = ops.A.attention(s[0], s[1], s[2], causal=True)
        return [o, lse, *ops.A.attention_backward(s[0], s[1], s[2], o, lse, s[3], causal=True)]

    def state(seed):
        return [up(ops, x) for x in attention_case(seed, (1, 1200, 900, 4, 2, 64))]

    states = [state(seed) for seed in (50, 60)]
    want = [bits(call(s)) for s in states]
    torch.cuda.synchronize()
    graphs = []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(s)
        graphs.append((g, out))
    for turn in range(4):
        for (g, out), ref in zip(graphs, want):
            for o in out:
                o.storage.fill_(7.0)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(bits(out), ref)), turn
        call(state(70 + turn))
        torch.cuda.synchronize()
    for g, _ in graphs:  # one behind the other, without a wait between them
        g.replay()
    torch.cuda.synchronize()
    for (_, out), ref in zip(graphs, want):
        assert all(torch.equal(x, y) for x, y in zip(bits(out), ref))


def test_a_workspace_that_is_too_small_is_refused(ops):
    import ctypes as C

    from tenmo_amd import _transformer

    L = _transformer.load()
    x = up(ops, randn(1, 3000, 64))
    v = C.byref(x.c_view())
    p = x.data_ptr()
    need = L.tenmo_hip_layer_norm_backward_workspace_bytes(3000, 64)
    for ws, size in ((p, need - 1), (None, need)):
        assert L.tenmo_hip_layer_norm_backward_f32(v, p, p, p, p, None, p, None, 0, ws, size, 0) == -3 and b"workspace" in L.tenmo_hip_last_error()
    assert L.tenmo_hip_layer_norm_backward_f32(v, p, p, p, p, None, p, None, 0, p + 4, need, 0) == -3 and b"aligned" in L.tenmo_hip_last_error()
    h = up(ops, randn(1, 300, 64))
    need = L.tenmo_hip_vocabulary_loss_forward_workspace_bytes(300, 64, 300)
    assert L.tenmo_hip_vocabulary_loss_forward_f32(C.byref(h.c_view()), C.byref(h.transpose().c_view()), None, p, 1, -100, 0.0, p, p, p, p, p, need - 1, 0) == -3
    q = up(ops, randn(1, 2, 400, 8, 64))
    qv = C.byref(q.c_view())
    need = L.tenmo_hip_attention_backward_workspace_bytes(2, 400, 400, 8, 8, 64)
    assert need > 0 and L.tenmo_hip_attention_backward_f32(qv, qv, qv, 0.1, 0, None, None, p, p, p, qv, None, None, 0, p, need - 1, 0) == -3


@pytest.mark.parametrize("wrong", ["shape", "dtype", "host", "reduction"])
def test_python_refusals(ops, wrong):
    from tenmo_amd import TenmoHipError

    h, w, t = up(ops, randn(1, 8, 4)), up(ops, randn(2, 4, 9)), torch.zeros(8, dtype=torch.int64, device="cuda")
    loss = ops.V.vocabulary_loss(h, w, None, t)
    with pytest.raises(TenmoHipError):
        if wrong == "shape":
            ops.V.vocabulary_loss(h, up(ops, randn(2, 5, 9)), None, t)
        elif wrong == "dtype":
            ops.V.vocabulary_loss(h, w, None, t.float())
        elif wrong == "host":
            ops.V.vocabulary_loss(h, w, None, t.cpu())
        else:
            ops.V.vocabulary_loss_backward(h, w, None, t, loss, torch.ones(1, device="cuda"), reduction="max")
