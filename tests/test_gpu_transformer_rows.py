"""Each row of a result on its own: attention's and the vocabulary loss's, where sizes within a call lie far apart.

A row is a sum of products.  Its error is measured against what enters it, the square root of the sum of the squares of its terms, so that neither the largest row of the call nor
terms that cancel count.  Tolerances are those of whole results in test_gpu_transformer.py, 1e-5 and 2e-5 for gradients: a term is off by the roundings of its factors (2^-22 as two halves,
2^-24 in fp32) and, where it holds a probability exp(-t), by that of its exponent, (t + 2 + |score|) 2^-24, which is 4e-6 at t = |score| = 32; the roundings of a sum have both signs.
"""
import math

import pytest
import torch

from helpers import RTOL_FRO
from test_gpu_transformer import down, ops, randn, up  # noqa: F401  (ops is a fixture)

pytestmark = pytest.mark.gpu


def rows_close(got, want, size, tol, what):
    """|got - want| of each row (the last axis) against its size."""
    got = got.double()
    assert bool(torch.isfinite(got).all()), what
    err = (got - want).norm(dim=-1)
    worst = torch.where(size > 0, err / size.clamp(min=1e-300), torch.where(err > 0, math.inf, 0.0))
    at = int(worst.argmax())
    print(f"{what}: {worst.max():.2e} in row {at}, median {worst.median():.2e}", flush=True)
    assert worst.max() <= tol, (what, at, float(worst.max()))


# ---- attention ----------------------------------------------------------------------------------------------------------------------


def attention_rows(q, k, v, scale, causal, dout):
    """out and gradients of one sequence [1, n, H, D] in 64 bits, each with the sizes of its rows."""
    n, m, group, D = q.shape[1], k.shape[1], q.shape[2] // k.shape[2], q.shape[3]
    q, k, v, dout = (t[0].double().transpose(0, 1) for t in (q, k, v, dout))
    kk, vv = (t.repeat_interleave(group, 0) for t in (k, v))
    s = scale * q @ kk.transpose(1, 2)
    if causal:
        s = s.masked_fill(torch.arange(m)[None, :] > torch.arange(n)[:, None] + m - n, -math.inf)
    p = torch.softmax(s, -1)
    o, dp = p @ vv, dout @ vv.transpose(1, 2)
    delta = (dout * o).sum(-1, keepdim=True)
    ds = p * (dp - delta) * scale
    dot = dout.norm(dim=-1, keepdim=True) * vv.norm(dim=-1)[:, None, :] / math.sqrt(D)  # the size of dp's own terms
    ds2 = (p * (dp.abs() + delta.abs() + dot) * scale) ** 2
    square = lambda t: (t ** 2).sum(-1, keepdim=True)  # noqa: E731
    shared = lambda t: t.reshape(k.shape[0], group, *t.shape[1:]).sum(1)  # noqa: E731
    want = [o, ds @ kk, shared(ds.transpose(1, 2) @ q), shared(p.transpose(1, 2) @ dout)]
    size = [(p ** 2) @ square(vv), ds2 @ square(kk), shared(ds2.transpose(1, 2) @ square(q)), shared((p ** 2).transpose(1, 2) @ square(dout))]
    return [t.transpose(0, 1)[None] for t in want], [t.transpose(0, 1)[None, ..., 0].sqrt() for t in size]


def check_attention(ops, q, k, v, dout, scale, causal):
    want, size = attention_rows(q, k, v, scale, causal, dout)
    Q, K, V, DO = (up(ops, t) for t in (q, k, v, dout))
    o, lse = ops.A.attention(Q, K, V, scale=scale, causal=causal)
    grads = ops.A.attention_backward(Q, K, V, o, lse, DO, scale=scale, causal=causal)
    rows_close(down(o), want[0], size[0], RTOL_FRO, "out")
    for g, w, s, what in zip(grads, want[1:], size[1:], ("grad_q", "grad_k", "grad_v")):
        rows_close(down(g), w, s, 2 * RTOL_FRO, what)


SIZES = [  # queries, keys, heads, kv_heads, dim, causal
    (600, 600, 4, 4, 64, True),
    (600, 600, 4, 2, 64, False),
    (333, 700, 8, 2, 128, True),
    (1100, 1000, 4, 4, 32, False),
    (400, 400, 6, 6, 80, True),
    (70, 70, 2, 2, 64, True),  # by rows
]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("where,factor", [("dout", 1e4), ("dout", 1e6), ("dout", 1e7), ("dout", 2.0 ** -10), ("dout", 2.0 ** -14), ("dout", 2.0 ** -20), ("dout", 2.0 ** -22), ("dout", 2.0 ** -40),
                                          ("dout", 1e-30), ("v", 1e4), ("v", 6e4), ("v", 2.0 ** -14), ("k", 2.0 ** -14), ("q", 2.0 ** -14), ("q", 2.0 ** -20)], ids=str)
@pytest.mark.parametrize("many", [False, True], ids=["one", "half"])
def test_attention_rows_of_different_sizes(ops, size, where, factor, many):  # noqa: F811
    """One row, or every row of the second half, times a factor: the others, and it, stay right by themselves."""
    n, m, H, Hk, D, causal = size
    t = {"q": randn(1, 1, n, H, D), "k": randn(2, 1, m, Hk, D), "v": randn(3, 1, m, Hk, D), "dout": randn(4, 1, n, H, D)}
    rows = t[where].shape[1]
    t[where][:, rows // 2 if many else rows // 3:rows if many else rows // 3 + 1] *= factor
    check_attention(ops, t["q"], t["k"], t["v"], t["dout"], 1.0 / math.sqrt(D), causal)


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("far", [8, 14, 18, 22, 30])
def test_attention_keys_of_little_weight(ops, size, far):  # noqa: F811
    """Keys that no query gives more than about e^-far: their gradients are sums of such probabilities alone."""
    n, m, H, Hk, D, causal = size
    q, k, v, dout = randn(5, 1, n, H, D), randn(6, 1, m, Hk, D), randn(7, 1, m, Hk, D), randn(8, 1, n, H, D)
    scale = 1.0 / math.sqrt(D)
    q[..., 0] = 3.0
    k[:, 1::3, :, 0] = -far / (3.0 * scale)
    check_attention(ops, q, k, v, dout, scale, causal)


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("seed", [0, 1])
def test_attention_values_far_out_of_little_weight(ops, size, seed):  # noqa: F811
    """Values 2^15 times the others' at keys of so little weight that they do not make the result: what is lost of their probabilities would show in it."""
    n, m, H, Hk, D, causal = size
    q, k, v, dout = randn(9 + seed, 1, n, H, D), randn(19 + seed, 1, m, Hk, D), randn(29 + seed, 1, m, Hk, D), randn(39 + seed, 1, n, H, D)
    scale = 1.0 / math.sqrt(D)
    q[..., 0] = 3.0
    v[:, 1::9] *= 2.0 ** 13
    k[:, 1::9, :, 0] = -22.0 / (3.0 * scale)
    check_attention(ops, q, k, v, dout, scale, causal)


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("small", [1.0, 2.0 ** -12, 2.0 ** -20, 2.0 ** -30], ids=str)
def test_attention_output_gradients_of_zeros(ops, size, small):  # noqa: F811
    """Queries without a gradient among others whose gradients are small against the first one's, which sees other keys: keys get theirs from the small ones alone."""
    n, m, H, Hk, D, causal = size
    q, k, v, dout = randn(101, 1, n, H, D), randn(102, 1, m, Hk, D), randn(103, 1, m, Hk, D), randn(104, 1, n, H, D)
    dout[:, 1:] *= small
    dout[:, 1::2] = 0.0
    q[:, 0] = 0.0
    q[:, 0, :, 0], k[:, -m // 3:, :, 0] = 8.0, -32.0  # (without a mask: the first query gives the last keys little)
    check_attention(ops, q, k, v, dout, 1.0 / math.sqrt(D), causal)


# ---- vocabulary loss ------------------------------------------------------------------------------------------------------------------


def vocabulary_rows(h, w, bias, target, upstream, reduction, smoothing):
    """Gradients in 64 bits with the sizes of their rows: of dH a token's, of dW a word's, of db a word's value."""
    h, w, bias = h.double(), w.double(), bias.double()
    x = h @ w + bias
    valid = target >= 0
    g = torch.softmax(x, -1) - smoothing / w.shape[1]
    g[torch.arange(len(target)), target.clamp(min=0)] -= 1.0 - smoothing
    s = upstream.double() / (valid.sum() if reduction == "mean" else 1)
    g = g * torch.where(valid, s, 0.0).expand(len(target))[:, None]
    square = lambda t, d: (t ** 2).sum(d)  # noqa: E731
    return [g @ w.t(), (h.t() @ g).t(), g.sum(0)[:, None]], [((g ** 2) @ square(w, 0)).sqrt(), ((g ** 2).t() @ square(h, 1)).sqrt(), g.abs().sum(0)], g.abs().t() @ h.norm(dim=1)


def check_vocabulary(ops, h, w, bias, target, upstream, reduction, smoothing, tied, one_way=None):
    want, size, magnitudes = vocabulary_rows(h, w, bias, target, upstream, reduction, smoothing)
    if one_way is not None:
        size[1] = magnitudes
    H, B, W = up(ops, h), up(ops, bias), up(ops, w.t().contiguous()).transpose() if tied else up(ops, w)
    kind = dict(ignore_index=-100, label_smoothing=smoothing)
    t = target.cuda()
    loss = ops.V.vocabulary_loss(H, W, B, t, **kind)
    gh, gw, gb = ops.V.vocabulary_loss_backward(H, W, B, t, loss, upstream.cuda(), reduction=reduction, **kind)
    # db sums probabilities of one sign, whose errors have one sign too where they are the exponent's: log2(e) as a float is off by 1.3e-8 of itself, so that every exp(-t) is by t 1.3e-8, 7e-7 at
    # t = 53, all in one direction.  Over 1500 tokens that alone is sqrt(1500) * 7e-7 = 2.7e-5 of the square root of the sum of squares: it is measured against the sum of magnitudes.
    for g, want_g, s, what in zip((down(gh), down(gw).t(), down(gb)[:, None]), want, size, ("grad_h", "grad_w", "grad_bias")):
        rows_close(g, want_g, s, 2 * RTOL_FRO + (one_way or 0.0), what)


VOCABULARY = [(300, 96, 20000), (700, 130, 9000), (1500, 64, 4100), (40, 96, 3000)]  # tokens, dim, words; the last by the kernels for few tokens


@pytest.mark.parametrize("size", VOCABULARY, ids=str)
@pytest.mark.parametrize("tied", [True, False], ids=["tied", "plain"])
@pytest.mark.parametrize("far", [8.0, 16.0, 20.0, 25.0, 40.0])
def test_vocabulary_words_of_little_weight(ops, size, tied, far):  # noqa: F811
    """A confident head: words whose logits lie `far` below the others' and that no target names.  Their rows of dW are sums of such probabilities alone."""
    m, d, v = size
    h, w, bias = randn(50, m, d), randn(51, d, v) * (1.3 / math.sqrt(d)), randn(52, v) * 0.1
    rare = torch.rand(v, generator=torch.Generator().manual_seed(53)) < 0.5
    rare[300:700] = True  # (and whole tiles of them)
    bias[rare] -= far
    common = torch.nonzero(~rare)[:, 0]
    target = common[torch.randint(0, len(common), (m,), generator=torch.Generator().manual_seed(54))]
    target[::17] = -100
    check_vocabulary(ops, h, w, bias, target, torch.ones(1), "mean", 0.0, tied)


@pytest.mark.parametrize("size", VOCABULARY, ids=str)
@pytest.mark.parametrize("tied", [True, False], ids=["tied", "plain"])
@pytest.mark.parametrize("what", ["upstream", "hidden", "both", "large"])
def test_vocabulary_tokens_of_different_sizes(ops, size, tied, what):  # noqa: F811
    """Tokens whose upstream gradients or hidden states lie up to 10^8 apart: a word that matters to small ones alone keeps its row of dW."""
    m, d, v = size
    h, w, bias = randn(60, m, d), randn(61, d, v) * (1.3 / math.sqrt(d)), randn(62, v) * 0.1
    target = torch.randint(0, v, (m,), generator=torch.Generator().manual_seed(63))
    target[::19] = -100
    upstream = randn(64, m)
    spread = 10.0 ** (-8.0 * torch.rand(m, generator=torch.Generator().manual_seed(65)))
    if what in ("upstream", "both"):
        upstream *= spread
    if what in ("hidden", "both"):
        h *= spread[:, None]
    if what == "large":
        upstream *= 1e25
        h *= 1e-25
    upstream[5] = 0.0
    bias[target.clamp(min=0)] -= 25.0  # (so that its tokens' G is nearly all that there is of a word)
    check_vocabulary(ops, h, w, bias, target, upstream, "none", 0.0, tied)


@pytest.mark.parametrize("size", VOCABULARY, ids=str)
@pytest.mark.parametrize("tied", [True, False], ids=["tied", "plain"])
@pytest.mark.parametrize("hidden", [1e-5, 1.0, 300.0])
def test_vocabulary_hidden_states_of_zeros(ops, size, tied, hidden):  # noqa: F811
    """Tokens that count, with hidden states of zeros: the weight's gradient is that of the tokens beside them."""
    m, d, v = size
    h, w, bias = randn(70, m, d) * hidden, randn(71, d, v) * (1.3 / math.sqrt(d) / hidden), randn(72, v) * 0.1
    h[::3] = 0.0
    target = torch.randint(0, v, (m,), generator=torch.Generator().manual_seed(73))
    target[::19] = -100
    check_vocabulary(ops, h, w, bias, target, torch.ones(1), "mean", 0.0, tied)


@pytest.mark.parametrize("m", [1000, 4100])
@pytest.mark.parametrize("tied", [True, False], ids=["tied", "plain"])
@pytest.mark.parametrize("near,far", [(0.0, 15.0), (0.3, 18.0), (2.0, 19.0), (4.5, 22.0), (8.6, 26.4)], ids=str)
def test_vocabulary_a_word_that_one_token_sees(ops, m, tied, near, far):  # noqa: F811
    """Words that one token gives a probability e^-near times the others' and all other tokens e^-far, with hidden states that point one way: what thousands of those add up to counts beside it.

    Terms of one sign, so rows of dW are measured against the sum of their magnitudes: a sum of n of them takes 3 n / 16 matrix instructions, each of which rounds it by up to 2^-24 of itself, 1.7e-6 of
    itself over 4100 tokens were they independent, and the sum is 64 times the square root of the sum of squares.  For the words that one token sees the two measures are the same to 1e-3.
    Their row is one probability, as good as that token's logit, in which 2 (near - far) meets a bias of as much: two operands held to 2^-22 and the product of their rests left out, 3 * 2^-22 of that, two
    additions of 2^-24."""
    d, v = 64, 2100
    h, w, bias = randn(80, m, d) * 0.3, randn(81, d, v) * 0.05, randn(82, v) * 0.1
    rare = torch.arange(v) % 3 == 0
    h[:, 0], h[m // 2, 0] = 3.0, 2.0
    h[:, 1] = 2.0
    w[0] = torch.where(rare, near - far, 0.0)
    w[1] = 0.0
    bias += torch.where(rare, 2.0 * (far - near) - near, 0.0)  # 3 (near - far) + this: -far; 2 (near - far) + this: -near
    target = torch.randint(0, v // 3, (m,), generator=torch.Generator().manual_seed(83)) * 3 + 1
    check_vocabulary(ops, h, w, bias, target, torch.ones(1), "mean", 0.0, tied, one_way=2.0 * (far - near) * (3 * 2.0 ** -22 + 2 * 2.0 ** -24))
