"""The measured operators: what a transformer block has around its attention and its losses.

  embedding       a token's row of a table, scaled, plus its position's
  embedding_grad  a table's gradient, each row the sum of its tokens' gradients, into the store
  layer_norm      layer norm forward and backward, weight and bias gradients into the store
  dropout         dropout from a counter-based generator, no mask stored, plus a residual
  linear          a matrix product with bias, activation, dropout and residual

A case's plain values: the operator (`op`), its rows (`rows`: tokens), its columns (`cols`), a
table's rows (`vocab`), a linear layer's outputs (`outs`), the element type (`dtype`) and what
else the operator takes.  `own` selects the framework's operators, whose weights are a parameter
store's tensors; the plain forms beside them are elementary operations in 32 bits, rounded once
at the end.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5  # layer norm's
DROP = 0.1
STREAM = 7  # which of a model's dropouts
CONTEXT = 1024  # positions of a sequence
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # the token just generated, on its way into GPT-2 124M: the smallest call, all latency
        dict(name="embedding_one_token", op="embedding", rows=1, cols=768, vocab=50257,
             dtype="bf16", scaled=False, positions=True),
        # sixteen sequences of 1024 tokens into GPT-2 124M
        dict(name="embedding_batch", op="embedding", rows=16384, cols=768, vocab=50257,
             dtype="bf16", scaled=False, positions=True),
        # the character model in full precision, two micro-batches: few rows that many tokens share
        dict(name="embedding_grad_char", op="embedding_grad", rows=4099, cols=384, vocab=65,
             dtype="fp32", scaled=True, micro=2),
        # GPT-2 124M's table from sixteen sequences of 1024 tokens
        dict(name="embedding_grad_124m", op="embedding_grad", rows=16384, cols=768, vocab=50257,
             dtype="bf16", scaled=False, micro=1),
        # a character model's activation with an odd number of tokens: short, all latency
        dict(name="layer_norm_char_fp32", op="layer_norm", rows=257, cols=384, dtype="fp32",
             residual=False),
        # GPT-2 774M, eight sequences of 1024 tokens, the residual stream's gradient added
        dict(name="layer_norm_774m", op="layer_norm", rows=8192, cols=1280, dtype="bf16",
             residual=True),
        # an activation of odd width in full precision
        dict(name="dropout_odd_fp32", op="dropout", rows=1021, cols=1537, dtype="fp32",
             residual=False),
        # GPT-2 1558M's residual stream, sixteen sequences of 1024 tokens
        dict(name="dropout_1558m", op="dropout", rows=16384, cols=1600, dtype="bf16",
             residual=True),
        # one generated token's logits, by the tied table of GPT-2 124M
        dict(name="linear_one_token", op="linear", rows=1, cols=768, outs=50257, dtype="bf16",
             activation=None, bias=False, dropout=False, residual=False, transposed=True),
        # the character model's MLP in full precision, an odd number of tokens
        dict(name="linear_char_fp32", op="linear", rows=3585, cols=384, outs=1536, dtype="fp32",
             activation="gelu", bias=True, dropout=False, residual=False, transposed=False),
        # GPT-2 774M's MLP, eight sequences of 1024 tokens: up, with GELU
        dict(name="linear_774m_up", op="linear", rows=8192, cols=1280, outs=5120, dtype="bf16",
             activation="gelu_tanh", bias=True, dropout=False, residual=False, transposed=False),
        # and down, back onto the residual stream
        dict(name="linear_774m_down", op="linear", rows=8192, cols=5120, outs=1280, dtype="bf16",
             activation=None, bias=True, dropout=True, residual=True, transposed=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the same ranges: one row to 16384, from the character model's sizes to
    GPT-2 1558M's, no larger than the largest listed one of its operator's kind."""
    op = rng.choice(["embedding", "embedding_grad", "layer_norm", "dropout", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    while True:
        c = dict(op=op, rows=_log_int(rng, 1, 16384), cols=_log_int(rng, 33, 6400), dtype=dtype)
        if op in ("embedding", "embedding_grad"):
            c.update(vocab=_log_int(rng, 65, 131072), scaled=rng.random() < 0.5)
            if c["vocab"] * c["cols"] > 50257 * 768 or c["rows"] * c["cols"] > 16384 * 768:
                continue
            if op == "embedding":
                c.update(positions=rng.random() < 0.5)
            else:
                c.update(micro=rng.choice([1, 1, 2]))
            return c
        if op in ("layer_norm", "dropout"):
            c.update(residual=rng.random() < 0.5)
            if c["rows"] * c["cols"] > (8192 * 1280 if op == "layer_norm" else 16384 * 1600):
                continue
            return c
        c.update(outs=_log_int(rng, 33, 6400), activation=rng.choice([None, "gelu", "gelu_tanh"]),
                 bias=rng.random() < 0.7, dropout=rng.random() < 0.3, residual=rng.random() < 0.4,
                 transposed=rng.random() < 0.5)
        # (a product in full precision takes several of the matrix instructions)
        if c["rows"] * c["cols"] * c["outs"] > 8192 * 1280 * 5120 // (6 if dtype == "fp32" else 1):
            continue
        return c


# ---- inputs -----------------------------------------------------------------------------------
def _tokens(rows, vocab, gen):
    """A text's tokens: the k-th most frequent about 1 / k as often as the first, frequent ones
    anywhere in the table; a few places are padding."""
    rank = torch.exp(torch.rand(rows, generator=gen, device="cuda") * math.log(vocab + 1)) - 1
    order = torch.randperm(vocab, generator=gen, device="cuda")
    t = order[rank.long().clamp(0, vocab - 1)]
    if rows > 16:
        t[torch.rand(rows, generator=gen, device="cuda") < 0.02] = -1
    return t


def _activation(rows, cols, dtype, gen):
    """What a residual stream looks like: a few channels far larger than the rest, off centre."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    channel = torch.exp(0.7 * torch.randn(cols, generator=gen, device="cuda"))
    return (x * channel + 0.2).to(dtype)


def _gradient(rows, cols, dtype, gen):
    return (torch.randn(rows, cols, generator=gen, device="cuda") * 1e-3).to(dtype)


def _weights(c, dtype, gen):
    """The store's tensors, as a trained model has them."""
    op = c["op"]

    def normal(shape, std, mean=0.0):
        return (torch.randn(shape, generator=gen, device="cuda") * std + mean).to(dtype)

    if op in ("embedding", "embedding_grad"):
        table = normal((c["vocab"], c["cols"]), 0.14)
        return [table, normal((CONTEXT, c["cols"]), 0.02)] if c.get("positions") else [table]
    if op == "layer_norm":
        return [normal((c["cols"],), 0.2, 1.0), normal((c["cols"],), 0.1)]
    if op == "linear":
        shape = (c["outs"], c["cols"]) if c["transposed"] else (c["cols"], c["outs"])
        return [normal(shape, c["cols"] ** -0.5), normal((c["outs"],), 0.1)]
    return [normal((64,), 1.0)]


def prepare(case, seed):
    c, op = case, case["op"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, rows, cols = TYPES[c["dtype"]], c["rows"], c["cols"]
    s = {"case": c, "seed": seed * 2654435761 % 2 ** 63, "w": _weights(c, dtype, gen)}
    if op in ("embedding", "embedding_grad"):
        micro = c.get("micro", 1)
        s["tokens"] = [_tokens(rows, c["vocab"], gen) for _ in range(micro)]
        if op == "embedding_grad":
            s["dy"] = [_gradient(rows, cols, dtype, gen) for _ in range(micro)]
        elif c["positions"]:
            s["positions"] = (torch.arange(rows, device="cuda") + seed % 97) % CONTEXT
    else:
        s["x"] = _activation(rows, cols, dtype, gen)
        if op == "layer_norm":
            s["dy"] = _gradient(rows, cols, dtype, gen)
        width = c["outs"] if op == "linear" else cols
        s["residual"] = None
        if c["residual"]:
            s["residual"] = _gradient(rows, cols, dtype, gen) if op == "layer_norm" else \
                _activation(rows, width, dtype, gen)
    if own:  # what a training program keeps: its parameter store
        s["store"] = _store(c, s["w"])
    return s


def _store(c, weights):
    """The store of the operator's weights, in the precision of the case, on torch's stream."""
    import os
    import sys
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tt-perf_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ttperf
    store = ttperf.ParamStore([tuple(w.shape) for w in weights],
                              mode="fp32" if c["dtype"] == "fp32" else "mixed")
    store.set_stream(torch.cuda.current_stream())
    for i, w in enumerate(weights):
        store.upload(ttperf.BUF_MASTER, i, w.float().reshape(-1))
    return store


# ---- one pass ---------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _scale(c):
    return math.sqrt(c["cols"]) if c["scaled"] else 1.0


def _run_own(s):
    c, op, store = s["case"], s["case"]["op"], s["store"]
    if op == "embedding":
        if c["positions"]:
            return store.embedding(0, s["tokens"][0], scale=_scale(c), position=1,
                                   positions=s["positions"])
        return store.embedding(0, s["tokens"][0], scale=_scale(c))
    if op == "embedding_grad":
        store.zero_grad(set_to_none=True, fill=False)
        for tokens, dy in zip(s["tokens"], s["dy"]):
            store.accumulate_embedding_grad(0, tokens, dy, scale=_scale(c))
        return _gradients(s, 1)[0].reshape(-1)
    if op == "layer_norm":
        store.zero_grad(set_to_none=True, fill=False)
        r = store.layer_norm(0, s["x"], bias=1, eps=EPS)
        dx = store.layer_norm_backward(0, s["x"], s["dy"], r.mean, r.rstd, bias=1,
                                       add=s["residual"])
        dw, db = _gradients(s, 2)
        return {"y": r.y, "dx": dx, "dw": dw, "db": db}
    if op == "dropout":
        return store.dropout(s["x"], DROP, s["seed"], stream=STREAM, residual=s["residual"])
    return store.linear(0, s["x"], bias=1 if c["bias"] else None, activation=c["activation"],
                        dropout=(DROP, s["seed"], STREAM) if c["dropout"] else None,
                        residual=s["residual"], transposed=c["transposed"])


def _gradients(s, n):
    """torch views of the store's gradients, made once."""
    if "views" not in s:
        import ttperf
        s["views"] = [s["store"].tensors[i].torch_view(ttperf.BUF_GRAD) for i in range(n)]
    return s["views"]


def _run_plain(s):
    c, op, w = s["case"], s["case"]["op"], s["w"]
    dtype = TYPES[c["dtype"]]
    if op == "embedding":
        y = _plain_rows(w[0], s["tokens"][0]) * _scale(c)
        if c["positions"]:
            y = y + _plain_rows(w[1], s["positions"])
        return y.to(dtype)
    if op == "embedding_grad":
        total = None
        for tokens, dy in zip(s["tokens"], s["dy"]):
            g = torch.zeros(c["vocab"] + 1, c["cols"], device="cuda")  # the last row: padding
            g.index_add_(0, torch.where(tokens >= 0, tokens, c["vocab"]), dy.float() * _scale(c))
            # each micro-batch is rounded to the gradients' type
            total = (g[:-1] if total is None else total.float() + g[:-1]).to(dtype)
        return total.reshape(-1)
    x = s["x"].float()
    if op == "layer_norm":
        dy = s["dy"].float()
        d = x - x.mean(1, keepdim=True)
        r = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
        h = d * r
        g = dy * w[0].float()
        dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
        if s["residual"] is not None:
            dx = dx + s["residual"].float()
        return {"y": (h * w[0].float() + w[1].float()).to(dtype), "dx": dx.to(dtype),
                "dw": (dy * h).sum(0).to(dtype), "db": dy.sum(0).to(dtype)}
    if op == "dropout":
        y = _plain_dropout(x, s["seed"])
    else:
        m = w[0].float()
        y = torch.mm(x, m.t() if c["transposed"] else m)
        if c["bias"]:
            y = y + w[1].float()
        if c["activation"] == "gelu":
            y = y * (0.5 * (1 + torch.erf(y / math.sqrt(2))))
        elif c["activation"] == "gelu_tanh":
            y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
        if c["dropout"]:
            y = _plain_dropout(y, s["seed"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(dtype)


def _plain_rows(table, at):
    """The table's rows, 0 where there is no token."""
    return torch.where((at >= 0)[:, None], table[at.clamp(min=0)].float(), 0.0)


def _plain_dropout(y, seed):
    """Philox 4x32 of ten rounds (Salmon, Moraes, Dror and Shaw, 2011) on a counter of 8 columns
    of a row: 16 bits an element, dropped below the threshold."""
    rows, cols = y.shape
    groups = -(-cols // 8)
    low = 0xFFFFFFFF
    g = torch.arange(rows * groups, device=y.device)
    c0, c1 = g & low, g >> 32
    c2, c3 = torch.full_like(g, STREAM), torch.zeros_like(g)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # (64 bits, whose sign does not matter)
        c0, c1, c2, c3 = (b >> 32 & low) ^ c1 ^ k0, b & low, (a >> 32 & low) ^ c3 ^ k1, a & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    words = torch.stack([c0, c1, c2, c3], 1)
    halves = torch.stack([words & 0xFFFF, words >> 16], 2).view(rows, groups * 8)[:, :cols]
    t = round(DROP * 65536)
    return torch.where(halves >= t, y * (65536 / (65536 - t)), 0.0)


# ---- the definitions in 64 bits ---------------------------------------------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)
    op, w = c["op"], [t.double() for t in s["w"]]
    if op == "embedding":
        tokens = s["tokens"][0]
        y = w[0][tokens.clamp(min=0)] * (_scale(c) * (tokens >= 0).double()[:, None])
        return y + w[1][s["positions"]] if c["positions"] else y
    if op == "embedding_grad":
        out = torch.zeros(c["vocab"], c["cols"], dtype=torch.float64, device="cuda")
        for tokens, dy in zip(s["tokens"], s["dy"]):
            live = tokens >= 0
            out.index_put_((tokens[live],), dy[live].double() * _scale(c), accumulate=True)
        return out.reshape(-1)
    x = s["x"].double()
    if op == "layer_norm":
        dy = s["dy"].double()
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        std = torch.sqrt(var + EPS)
        h = (x - mean) / std
        g = dy * w[0]
        n = c["cols"]
        dx = (g - (g.sum(1, keepdim=True) + h * (g * h).sum(1, keepdim=True)) / n) / std
        if s["residual"] is not None:
            dx += s["residual"].double()
        return {"y": torch.addcmul(w[1], h, w[0]), "dx": dx, "dw": (dy * h).sum(0),
                "db": dy.sum(0)}
    if op == "dropout":
        y = x
    else:
        y = x @ w[0].t() if c["transposed"] else x @ w[0]
        if c["bias"]:
            y += w[1]
        if c["activation"] == "gelu":
            y = y * torch.special.ndtr(y)
        elif c["activation"] == "gelu_tanh":
            y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
    if op == "dropout" or c["dropout"]:
        y = y * _exact_keep(y.shape[0], y.shape[1], s["seed"]).cuda()
    if s["residual"] is not None:
        y = y + s["residual"].double()
    return y


def _exact_keep(rows, cols, seed):
    """0 or the kept elements' factor, from unsigned numbers on the host."""
    groups = (cols + 7) // 8
    mask, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    n = np.arange(rows * groups, dtype=np.uint64)
    x = [n & mask, n >> sh, np.full_like(n, STREAM), np.zeros_like(n)]
    keys = [np.uint64(seed % 2 ** 32), np.uint64(seed // 2 ** 32)]
    for r in range(10):
        p, q = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(q >> sh) ^ x[1] ^ keys[0], q & mask, (p >> sh) ^ x[3] ^ keys[1], p & mask]
        keys = [(keys[0] + np.uint64(0x9E3779B9)) & mask, (keys[1] + np.uint64(0xBB67AE85)) & mask]
    halves = np.stack([v for word in x for v in (word & np.uint64(0xFFFF), word >> np.uint64(16))],
                      axis=1).reshape(rows, groups * 8)[:, :cols]
    t = int(DROP * 65536 + 0.5)
    return torch.from_numpy((halves >= t) * (65536 / (65536 - t)))


# ---- what a pass cannot do without ------------------------------------------------------------
def work(case):
    """Bytes: each input read once, each output written once (of a table the rows that are looked
    up; a gradient's table whole, and its touched rows again for a second micro-batch).
    Operations: 12 per layer norm element and direction, 20 per random element, 2 per product."""
    c, op, rows, cols = case, case["op"], case["rows"], case["cols"]
    size = 2 if c["dtype"] == "bf16" else 4
    n = rows * cols
    if op == "embedding":
        looked_up = min(rows, c["vocab"]) + (min(rows, CONTEXT) if c["positions"] else 0)
        ids = rows * (16 if c["positions"] else 8)
        return {"bytes": (n + looked_up * cols) * size + ids, "flops": 2 * n}
    if op == "embedding_grad":
        again = (c["micro"] - 1) * 2 * min(rows, c["vocab"]) * cols
        return {"bytes": (c["micro"] * n + c["vocab"] * cols + again) * size + c["micro"] * rows * 8,
                "flops": 2 * c["micro"] * n}
    if op == "layer_norm":  # x, y; x again, dy, dx (and the residual's); mean and rstd twice
        return {"bytes": (5 + c["residual"]) * n * size + 4 * cols * size + 16 * rows,
                "flops": 24 * n}
    if op == "dropout":
        return {"bytes": (2 + c["residual"]) * n * size, "flops": 20 * n}
    m = c["outs"]
    return {"bytes": (n + cols * m + rows * m * (1 + c["residual"]) + m * c["bias"]) * size,
            "flops": 2 * n * m + rows * m * (20 if c["dropout"] or c["activation"] else 2)}
