"""Cases for the operators of a transformer's training step: layer norm, attention and the vocabulary loss.

Each case is one call as a program makes it: the forward call alone (evaluation, a decoded token), or the forward call followed by the
backward call on the same inputs ("train").  Everything is fp32, the library's type.  ``run`` computes a case in elementary torch
operations, or through ``tenmo_amd`` where ``own`` is set; ``exact`` computes it in 64 bits through torch's autograd.
"""
import math

import torch

own = False

NORM, ATTENTION, VOCABULARY = "layer_norm", "attention", "vocabulary"


def _norm(name, rows, width, train=True, affine=True):
    return {"name": name, "op": NORM, "rows": rows, "width": width, "train": train, "affine": affine}


def _attention(name, batch, queries, keys, heads, kv_heads, dim, causal, train, ragged="none"):
    return {"name": name, "op": ATTENTION, "batch": batch, "queries": queries, "keys": keys, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "causal": causal, "train": train, "ragged": ragged}


def _vocabulary(name, tokens, dim, vocabulary, train, reduction="mean", smoothing=0.0, tied=True, bias=False):
    return {"name": name, "op": VOCABULARY, "tokens": tokens, "dim": dim, "vocabulary": vocabulary, "train": train, "reduction": reduction,
            "smoothing": smoothing, "tied": tied, "bias": bias}


def listed():
    return [
        # the norm in front of a block while one sequence decodes: launch latency alone
        _norm("norm_one_token", 1, 768, train=False),
        # a GPT-2 sized training batch (8 sequences of 1024 tokens), the size the library's linears are benchmarked at
        _norm("norm_gpt2_train", 8192, 768),
        # an odd width (no 16-byte rows) and many rows, past the caches
        _norm("norm_odd_train", 30011, 2049),
        # one new token for each of 32 sequences against a cache of up to 4096 positions, every sequence of its own length
        _attention("attention_decode", 32, 1, 4096, 12, 12, 64, False, False, "lengths"),
        # one new token of one long sequence, heads in groups: few rows, a long axis
        _attention("attention_decode_long", 1, 1, 65536, 32, 8, 128, False, False),
        # a short padded batch with an empty row, odd sizes: latency
        _attention("attention_small_train", 2, 33, 33, 4, 4, 32, False, True, "empty"),
        # GPT-2's attention over the training batch: the sizes of the library's attention-shaped products
        _attention("attention_gpt2_train", 8, 1024, 1024, 12, 12, 64, True, True),
        # a long sequence, wide heads in groups of four
        _attention("attention_long_train", 1, 8192, 8192, 16, 4, 128, True, True),
        # evaluation of padded prompts, a head width that is no power of two
        _attention("attention_prompt", 4, 777, 777, 16, 16, 80, True, False, "lengths"),
        # a small vocabulary (characters, bytes with merges) in a small model
        _vocabulary("vocabulary_small_train", 64, 128, 1000, True),
        # GPT-2's LM head over the training batch, weight tied to the embedding
        _vocabulary("vocabulary_gpt2_train", 8192, 768, 50257, True),
        # an odd head: untied weight with a bias, smoothing, summed
        _vocabulary("vocabulary_odd_train", 1001, 1030, 32003, True, "sum", 0.1, False, True),
    ]


def _spread(rng, low, high):
    """A whole number of low..high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _drawn(rng):
    op = rng.choice((NORM, ATTENTION, ATTENTION, VOCABULARY))
    if op == NORM:
        return _norm("", _spread(rng, 1, 32768), _spread(rng, 16, 8192), rng.random() < 0.7, rng.random() < 0.8)
    if op == ATTENTION:
        dim = rng.choice((32, 64, 80, 96, 128, rng.randint(8, 128)))
        group = rng.choice((1, 1, 2, 4, 8))
        kv_heads = rng.randint(1, 16 // group)
        if rng.random() < 0.35:  # decoding: a few new tokens against a cache
            queries = rng.choice((1, 1, 1, rng.randint(2, 8)))
            return _attention("", _spread(rng, 1, 32), queries, max(queries, _spread(rng, 16, 65536)), kv_heads * group, kv_heads, dim, queries > 1, False,
                              rng.choice(("none", "lengths")))
        train = rng.random() < 0.6
        least = 8 if train else 1  # a lone key has probability one: its gradients to q and k are zero, and rounding is all there is to compare
        n = _spread(rng, least, 8192)
        keys = n if rng.random() < 0.8 else _spread(rng, least, 8192)
        return _attention("", _spread(rng, 1, 16), n, keys, kv_heads * group, kv_heads, dim, keys >= n and rng.random() < 0.7, train,
                          rng.choice(("none", "lengths", "empty")))
    return _vocabulary("", _spread(rng, 1, 8192), _spread(rng, 32, 1600), _spread(rng, 300, 60000), rng.random() < 0.7,
                       rng.choice(("mean", "sum", "none")), rng.choice((0.0, 0.1)), rng.random() < 0.6, rng.random() < 0.4)


def draw(rng):
    flops = max(work(c)["flops"] for c in listed())
    elements = max(_elements(c) for c in listed())
    while True:
        case = _drawn(rng)
        if work(case)["flops"] <= flops and _elements(case) <= elements:
            del case["name"]
            return case


def _elements(case):
    """Values that the plain form holds at once, about."""
    if case["op"] == NORM:
        return case["rows"] * case["width"]
    if case["op"] == ATTENTION:
        return case["batch"] * (case["heads"] * case["queries"] * case["keys"] + case["kv_heads"] * case["keys"] * case["dim"])
    return case["tokens"] * case["vocabulary"] + case["dim"] * case["vocabulary"]


# ---- inputs -------------------------------------------------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale

    if case["op"] == NORM:
        rows, width = case["rows"], case["width"]
        s["eps"] = 1e-5
        s["x"] = normal(rows, width, scale=1.5) + 0.3
        s["weight"] = 1.0 + normal(width, scale=0.1) if case["affine"] else None
        s["bias"] = normal(width, scale=0.1) if case["affine"] else None
        s["dy"] = normal(rows, width) if case["train"] else None
    elif case["op"] == ATTENTION:
        b, n, m, h, hk, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
        s["scale"] = 1.0 / math.sqrt(d)
        s["q"], s["k"], s["v"] = normal(b, n, h, d), normal(b, m, hk, d), normal(b, m, hk, d)
        s["dout"] = normal(b, n, h, d) if case["train"] else None
        s["lengths"] = s["starts"] = None
        if case["ragged"] != "none":
            lengths = torch.randint(max(1, m // 2), m + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
            if case["ragged"] == "empty":
                lengths[seed % b] = 0
            s["lengths"] = lengths
            if n < m:  # new tokens at the end of each sequence
                s["starts"] = lengths - n
    else:
        m, d, v = case["tokens"], case["dim"], case["vocabulary"]
        w = normal(v, d, scale=1.3 / math.sqrt(d))
        s["w"] = w if case["tied"] else w.t().contiguous()  # tied: the embedding [vocabulary, dim], used transposed
        s["h"] = normal(m, d)
        s["b"] = normal(v, scale=0.1) if case["bias"] else None
        s["ignore"] = -100
        target = torch.randint(0, v, (m,), generator=g, device="cuda", dtype=torch.int64)
        s["target"] = torch.where(torch.rand(m, generator=g, device="cuda") < 0.05, -100, target)
        s["upstream"] = (normal(m) if case["reduction"] == "none" else normal(1, scale=0.1) + 1.0) if case["train"] else None
    return s


# ---- the operators in their plain form ----------------------------------------------------------------------------------------------


def run(s):
    if own:
        return {NORM: _own_norm, ATTENTION: _own_attention, VOCABULARY: _own_vocabulary}[s["op"]](s)
    return {NORM: _plain_norm, ATTENTION: _plain_attention, VOCABULARY: _plain_vocabulary}[s["op"]](s)


def _plain_norm(s):
    x, w, b = s["x"], s["weight"], s["bias"]
    mean = x.mean(-1, keepdim=True)
    centred = x - mean
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + s["eps"])
    xhat = centred * rstd
    y = xhat * w + b if w is not None else xhat
    if not s["train"]:
        return {"y": y}
    dy = s["dy"]
    g = dy * w if w is not None else dy
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    out = {"y": y, "mean": mean[:, 0], "rstd": rstd[:, 0], "dx": dx}
    if w is not None:
        out["dw"], out["db"] = (dy * xhat).sum(0), dy.sum(0)
    return out


def _allowed(s, device):
    """[batch or 1, 1, queries, keys]: which keys a query sees; None where it sees all of them."""
    n, m = s["queries"], s["keys"]
    if not s["causal"] and s["lengths"] is None:
        return None
    j = torch.arange(m, device=device)
    ok = torch.ones(1, 1, n, m, dtype=torch.bool, device=device)
    if s["lengths"] is not None:
        ok = ok & (j < s["lengths"][:, None, None, None])
    if s["causal"]:
        start = s["starts"][:, None, None, None] if s["starts"] is not None else m - n
        ok = ok & (j <= torch.arange(n, device=device)[:, None] + start)
    return ok


def _plain_attention(s):
    b, n, m, h, hk, d = (s[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    q = s["q"].permute(0, 2, 1, 3)
    k, v = (s[x].permute(0, 2, 1, 3).repeat_interleave(h // hk, 1).contiguous() for x in ("k", "v"))
    scores = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    ok = _allowed(s, q.device)
    if ok is not None:
        scores = torch.where(ok, scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    p = torch.exp(scores - top)
    del scores
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    lse = (top + torch.log(total))[..., 0]
    o = torch.matmul(p, v)
    out = {"out": o.permute(0, 2, 1, 3).contiguous()}
    if not s["train"]:
        return out
    do = s["dout"].permute(0, 2, 1, 3)
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = p * (torch.matmul(do, v.transpose(2, 3)) - (do * o).sum(-1, keepdim=True)) * s["scale"]
    dk = torch.matmul(ds.transpose(2, 3), q)
    dq = torch.matmul(ds, k)
    dk, dv = (x.reshape(b, hk, h // hk, m, d).sum(2) for x in (dk, dv))
    out["lse"] = lse
    out["dq"], out["dk"], out["dv"] = (x.permute(0, 2, 1, 3).contiguous() for x in (dq, dk, dv))
    return out


def _plain_vocabulary(s):
    h, w, target, smoothing, n = s["h"], s["w"], s["target"], s["smoothing"], s["vocabulary"]
    w = w.t() if s["tied"] else w
    logits = torch.matmul(h, w)
    if s["b"] is not None:
        logits = logits + s["b"]
    valid = target != s["ignore"]
    t = torch.where(valid, target, 0)[:, None]
    top = logits.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(logits - top).sum(-1, keepdim=True))
    loss = (1.0 - smoothing) * (lse - logits.gather(1, t)) + smoothing * (lse - logits.mean(-1, keepdim=True))
    loss = torch.where(valid, loss[:, 0], 0.0)
    count = valid.sum()
    out = {"loss": loss, "loss_sum": loss.double().sum().float().reshape(1), "valid": count.int().reshape(1)}
    if not s["train"]:
        return out
    scale = {"mean": s["upstream"] / count.clamp(min=1), "sum": s["upstream"], "none": s["upstream"]}[s["reduction"]]
    scale = torch.where(valid, scale, 0.0)[:, None]
    g = torch.exp(logits - lse)
    del logits
    g = g - smoothing / n
    g.scatter_add_(1, t, torch.full_like(g[:, :1], smoothing - 1.0))
    g = g * scale
    out["lse"] = lse[:, 0]
    out["dh"] = torch.matmul(g, w.t())
    out["dw"] = torch.matmul(g.t(), h) if s["tied"] else torch.matmul(h.t(), g)
    if s["b"] is not None:
        out["db"] = g.sum(0)
    return out


# ---- the same through the framework --------------------------------------------------------------------------------------------------


def _buffer(t):
    from tenmo_amd.ndbuffer import NDBuffer

    return None if t is None else NDBuffer(t.view(-1), t.shape)


def _back(buffer):
    return buffer.storage.view(buffer.shape)


def _own_norm(s):
    from tenmo_amd.norm import layer_norm, layer_norm_backward

    x, w, b = _buffer(s["x"]), _buffer(s["weight"]), _buffer(s["bias"])
    if not s["train"]:
        return {"y": _back(layer_norm(x, w, b, s["eps"], statistics=False)[0])}
    y, mean, rstd = layer_norm(x, w, b, s["eps"])
    dx, dw, db = layer_norm_backward(x, w, mean, rstd, _buffer(s["dy"]))
    out = {"y": _back(y), "mean": _back(mean), "rstd": _back(rstd), "dx": _back(dx)}
    if w is not None:
        out["dw"], out["db"] = _back(dw), _back(db)
    return out


def _own_attention(s):
    from tenmo_amd.attention import attention, attention_backward

    q, k, v = _buffer(s["q"]), _buffer(s["k"]), _buffer(s["v"])
    mask = {"scale": s["scale"], "causal": s["causal"], "key_lengths": s["lengths"], "query_starts": s["starts"]}
    if not s["train"]:
        return {"out": _back(attention(q, k, v, statistics=False, **mask)[0])}
    o, lse = attention(q, k, v, **mask)
    dq, dk, dv = attention_backward(q, k, v, o, lse, _buffer(s["dout"]), **mask)
    return {"out": _back(o), "lse": _back(lse), "dq": _back(dq), "dk": _back(dk), "dv": _back(dv)}


def _own_vocabulary(s):
    from tenmo_amd.vocabulary import vocabulary_loss, vocabulary_loss_backward

    h, w, b = _buffer(s["h"]), _buffer(s["w"]), _buffer(s["b"])
    w = w.transpose() if s["tied"] else w
    kind = {"ignore_index": s["ignore"], "label_smoothing": s["smoothing"]}
    loss = vocabulary_loss(h, w, b, s["target"], **kind)
    out = {"loss": _back(loss.per_sample), "loss_sum": _back(loss.loss_sum), "valid": loss.valid_count}
    if not s["train"]:
        return out
    dh, dw, db = vocabulary_loss_backward(h, w, b, s["target"], loss, s["upstream"], reduction=s["reduction"], **kind)
    out["lse"], out["dh"] = _back(loss.lse), _back(dh)
    out["dw"] = _back(dw.transpose() if s["tied"] else dw)  # the gradient of a transposed view is laid out as what it views
    if s["b"] is not None:
        out["db"] = _back(db)
    return out


# ---- what they cannot do without -----------------------------------------------------------------------------------------------------


def work(case):
    if case["op"] == NORM:
        n, extra = case["rows"] * case["width"], 2 * case["width"] if case["affine"] else 0
        if not case["train"]:
            return {"bytes": 4.0 * (2 * n + extra), "flops": 8.0 * n}
        return {"bytes": 4.0 * (4 * n + 2 * extra + 2 * case["rows"]), "flops": 20.0 * n}
    if case["op"] == ATTENTION:
        b, n, m, h, hk, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
        keys = m if case["ragged"] == "none" else 0.75 * m
        pairs = b * h * (n * keys - (0.5 * n * (n - 1) if case["causal"] else 0))
        rows, cache = b * n * h * d, b * keys * hk * d
        if not case["train"]:
            return {"bytes": 4.0 * (2 * rows + 2 * cache), "flops": 4.0 * d * pairs}
        return {"bytes": 4.0 * (4 * rows + 4 * cache), "flops": 12.0 * d * pairs}
    m, d, v = case["tokens"], case["dim"], case["vocabulary"]
    if not case["train"]:
        return {"bytes": 4.0 * (m * d + v * d), "flops": 2.0 * m * d * v}
    return {"bytes": 8.0 * (m * d + v * d), "flops": 6.0 * m * d * v}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {NORM: _exact_norm, ATTENTION: _exact_attention, VOCABULARY: _exact_vocabulary}[s["op"]](s)


def _leaf(t):
    return None if t is None else t.double().requires_grad_(True)


def _exact_norm(s):
    x, w, b = _leaf(s["x"]), _leaf(s["weight"]), _leaf(s["bias"])
    var, mean = torch.var_mean(x, -1, correction=0)
    rstd = 1.0 / torch.sqrt(var + s["eps"])
    y = (x - mean[:, None]) * rstd[:, None]
    y = y * w + b if w is not None else y
    if not s["train"]:
        return {"y": y.detach()}
    y.backward(s["dy"].double())
    out = {"y": y.detach(), "mean": mean.detach(), "rstd": rstd.detach(), "dx": x.grad}
    if w is not None:
        out["dw"], out["db"] = w.grad, b.grad
    return out


def _exact_attention(s):
    q, k, v = (s[x].double().detach() for x in ("q", "k", "v"))
    group, m = s["heads"] // s["kv_heads"], s["keys"]
    out, lse = torch.zeros_like(q), torch.full((s["batch"], s["heads"], s["queries"]), float("-inf"), dtype=torch.float64, device=q.device)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    first = s["starts"].tolist() if s["starts"] is not None else [m - s["queries"]] * s["batch"]
    lengths = s["lengths"].tolist() if s["lengths"] is not None else [m] * s["batch"]
    piece = max(1, (1 << 26) // m)  # queries at a time
    for b in range(s["batch"]):
        n = lengths[b]
        if n <= 0:
            continue
        for h in range(s["heads"]):
            kh, vh = (x[b, :n, h // group].clone().requires_grad_(True) for x in (k, v))
            for lo in range(0, s["queries"], piece):
                qh = q[b, lo:lo + piece, h].clone().requires_grad_(True)
                x = (qh @ kh.T) * s["scale"]
                if s["causal"]:
                    last = first[b] + lo + torch.arange(qh.shape[0], device=x.device)[:, None]
                    x = x.masked_fill(torch.arange(n, device=x.device) > last, -1e300)
                    none = (last < 0)
                else:
                    none = torch.zeros(qh.shape[0], 1, dtype=torch.bool, device=x.device)
                o = (torch.softmax(x, -1) @ vh).masked_fill(none, 0.0)
                out[b, lo:lo + piece, h] = o.detach()
                lse[b, h, lo:lo + piece] = torch.logsumexp(x.detach(), -1).masked_fill(none[:, 0], float("-inf"))
                if s["train"]:
                    o.backward(s["dout"][b, lo:lo + piece, h].double())
                    dq[b, lo:lo + piece, h] = qh.grad
            if s["train"]:
                dk[b, :n, h // group] += kh.grad
                dv[b, :n, h // group] += vh.grad
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv} if s["train"] else {"out": out}


def _exact_vocabulary(s):
    w, b = _leaf(s["w"]), _leaf(s["b"])
    n, count = s["tokens"], int((s["target"] != s["ignore"]).sum())
    loss, lse, dh = [], [], []
    piece = max(1, (1 << 26) // s["vocabulary"])  # rows at a time
    for lo in range(0, n, piece):
        h, t = _leaf(s["h"][lo:lo + piece]), s["target"][lo:lo + piece]
        x = h @ (w.T if s["tied"] else w)
        x = x + b if b is not None else x
        each = torch.nn.functional.cross_entropy(x, t, ignore_index=s["ignore"], label_smoothing=s["smoothing"], reduction="none")
        loss.append(each.detach())
        lse.append(torch.logsumexp(x.detach(), -1))
        if s["train"]:
            up = s["upstream"].double()
            up = up[lo:lo + piece] if s["reduction"] == "none" else (up / max(1, count) if s["reduction"] == "mean" else up).expand(each.shape[0])
            each.backward(up)
            dh.append(h.grad)
    loss = torch.cat(loss)
    out = {"loss": loss, "loss_sum": loss.sum().reshape(1), "valid": None}
    if s["train"]:
        out.update(lse=torch.cat(lse), dh=torch.cat(dh), dw=w.grad)
        if b is not None:
            out["db"] = b.grad
    return out
