"""The measured operators: what a fine-tuning step has around the optimizer store.

  logprobs    each row's log-probability of its token, from logits (a reference model's scores)
  preference  the loss of chosen against rejected sequences, and the logits' gradient
  policy      the clipped policy loss with its KL term, and the logits' gradient
  checkpoint  an activation kept in 8 bits (blocks of 32 columns, power-of-two scales), restored
  gelu        GELU that keeps its input in 8 bits, forward and backward
  linear      a linear layer's input kept in 8 bits, and its weight and bias gradients from it,
              into the store's gradients

A case's plain values: the operator (`op`), its rows (`rows`: tokens), its columns (`vocab` of the
losses, `cols` of an activation, `outs` of a linear layer), the element type (`dtype`) and what
else the operator takes.  `own` selects the framework's operators; the plain forms beside them
are elementary operations in 32 bits, rounded once at the end.
"""
import math

import torch

own = False

BETA, SMOOTHING = 0.1, 0.05
CLIP_LOW, CLIP_HIGH, KL_COEF = 0.2, 0.28, 0.04
BLOCK = 32  # columns that share a scale
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one generated token's score over GPT-2's vocabulary: the smallest call, all latency
        dict(name="logprobs_one_token", op="logprobs", rows=1, vocab=50257, dtype="bf16",
             masked=0.0),
        # a reference model's scores of a batch of eight sequences of 1024 tokens
        dict(name="logprobs_batch", op="logprobs", rows=8192, vocab=50257, dtype="bf16",
             masked=0.1),
        # the character model (65 characters) in full precision: short rows, uneven sequences
        dict(name="preference_char", op="preference", rows=3001, vocab=65, dtype="fp32",
             masked=0.2, pairs=8, smoothing=0.0),
        # eight pairs of answers of about 600 tokens behind masked prompts, GPT-2's vocabulary
        dict(name="preference_gpt2", op="preference", rows=9733, vocab=50257, dtype="bf16",
             masked=0.3, pairs=8, smoothing=SMOOTHING),
        # a small rollout in full precision, no reference model
        dict(name="policy_rollout_fp32", op="policy", rows=1021, vocab=50257, dtype="fp32",
             masked=0.1, kl=0.0),
        # sixteen rollouts of 1024 tokens with a KL term: the largest loss
        dict(name="policy_gpt2", op="policy", rows=16384, vocab=50257, dtype="bf16", masked=0.15,
             kl=KL_COEF),
        # a character model's activation with an odd number of tokens, fp8 values
        dict(name="checkpoint_char_e4m3", op="checkpoint", rows=257, cols=384, dtype="fp32",
             fmt="e4m3"),
        # GPT-2 1558M's residual stream, sixteen sequences of 1024 tokens
        dict(name="checkpoint_1558m", op="checkpoint", rows=16384, cols=1600, dtype="bf16",
             fmt="int8"),
        # a hidden layer whose width is no multiple of a block, fp32, exact GELU
        dict(name="gelu_odd_fp32", op="gelu", rows=1003, cols=1537, dtype="fp32", fmt="int8",
             approximate="none"),
        # GPT-2 774M's hidden activation, eight sequences of 1024 tokens
        dict(name="gelu_774m", op="gelu", rows=8192, cols=5120, dtype="bf16", fmt="int8",
             approximate="tanh"),
        # the character model's MLP input in full precision: few tiles, many rows
        dict(name="linear_char_fp32", op="linear", rows=3585, cols=384, outs=1536,
             dtype="fp32", fmt="int8", transposed=False),
        # GPT-2 774M's MLP weight from eight sequences of 1024 tokens
        dict(name="linear_774m", op="linear", rows=8192, cols=1280, outs=5120, dtype="bf16",
             fmt="int8", transposed=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the same ranges: one row to 16384, from the character model's sizes to
    GPT-2 1558M's, no larger than the largest listed one of its operator's kind."""
    op = rng.choice(["logprobs", "preference", "policy", "checkpoint", "gelu", "linear"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    size = 2 if dtype == "bf16" else 4
    while True:
        rows = _log_int(rng, 1 if op == "logprobs" else 16, 16384)
        if op in ("logprobs", "preference", "policy"):
            c = dict(op=op, rows=rows, vocab=_log_int(rng, 65, 131072), dtype=dtype,
                     masked=rng.choice([0.0, 0.1, 0.3]))
            if rows * c["vocab"] * size > 1.2e9:
                continue
            if op == "preference":
                c.update(pairs=min(_log_int(rng, 1, 64), max(1, rows // 4)),
                         smoothing=rng.choice([0.0, SMOOTHING]))
            elif op == "policy":
                c.update(kl=rng.choice([0.0, KL_COEF]))
            return c
        c = dict(op=op, rows=rows, cols=_log_int(rng, 33, 6400), dtype=dtype,
                 fmt=rng.choice(["int8", "e4m3"]))
        if op == "gelu":
            c.update(approximate=rng.choice(["none", "tanh"]))
        elif op == "linear":
            c.update(outs=_log_int(rng, 33, 6400), transposed=rng.random() < 0.4)
            if rows * c["cols"] * c["outs"] > 8192 * 1280 * 5120 // (3 if dtype == "fp32" else 1):
                continue
        return c


# ---- inputs -----------------------------------------------------------------------------------
def _logits(c, gen):
    """What a language model's head gives: spread over the vocabulary, the token it was trained
    towards often well above the rest; some rows (prompts, padding) are masked."""
    rows, vocab, dtype = c["rows"], c["vocab"], TYPES[c["dtype"]]
    z = torch.randn(rows, vocab, generator=gen, device="cuda", dtype=dtype).mul_(2.5)
    y = torch.randint(vocab, (rows,), generator=gen, device="cuda")
    lift = torch.rand(rows, generator=gen, device="cuda") * 12
    z[torch.arange(rows, device="cuda"), y] += lift.to(dtype)
    hide = torch.rand(rows, generator=gen, device="cuda") < c["masked"]
    return z, torch.where(hide, -100, y)


def _near_logprobs(z, y, spread, gen):
    """Another model's log-probabilities of the tokens: near this one's."""
    parts = [torch.logsumexp(p.float(), 1) for p in z.split(1024)]
    logp = z.gather(1, y.clamp(min=0)[:, None])[:, 0].float() - torch.cat(parts)
    return logp + spread * torch.randn(len(logp), generator=gen, device="cuda")


def _starts(rows, sequences, gen):
    """Sequences of uneven length that share the rows out."""
    w = torch.rand(sequences, generator=gen, device="cuda") + 0.3
    ends = (torch.cumsum(w, 0) / w.sum() * rows).round().long()
    ends[-1] = rows
    return torch.cat([ends.new_zeros(1), ends])


def _activation(rows, cols, dtype, gen):
    """What a block's normalised input looks like: a few channels far larger than the rest."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    channel = torch.exp(0.7 * torch.randn(cols, generator=gen, device="cuda"))
    return (x * channel).to(dtype)


def prepare(case, seed):
    c, op = case, case["op"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[c["dtype"]]
    s = {"case": c}
    if op in ("logprobs", "preference", "policy"):
        s["z"], s["y"] = _logits(c, gen)
        if op == "preference":
            s["starts"] = _starts(c["rows"], 2 * c["pairs"], gen)
            s["ref"] = _near_logprobs(s["z"], s["y"], 0.05, gen)
        elif op == "policy":
            s["old"] = _near_logprobs(s["z"], s["y"], 0.15, gen)
            s["adv"] = torch.randn(c["rows"], generator=gen, device="cuda")
            s["ref"] = _near_logprobs(s["z"], s["y"], 0.2, gen) if c["kl"] else None
    else:
        s["x"] = _activation(c["rows"], c["cols"], dtype, gen)
        if op != "checkpoint":
            width = c["outs"] if op == "linear" else c["cols"]
            s["dy"] = (torch.randn(c["rows"], width, generator=gen, device="cuda") * 1e-3).to(dtype)
    if own:  # the handle that a training program keeps: its parameter store
        s["store"] = _store(c)
    return s


def _store(c):
    """The store of the layer's weight and bias (of one small tensor for the other operators), in
    the precision of the case, on torch's stream."""
    import os
    import sys
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tt-perf_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ttperf
    shapes = [(64,)]
    if c["op"] == "linear":
        weight = (c["outs"], c["cols"]) if c["transposed"] else (c["cols"], c["outs"])
        shapes = [weight, (c["outs"],)]
    store = ttperf.ParamStore(shapes, mode="fp32" if c["dtype"] == "fp32" else "mixed")
    store.set_stream(torch.cuda.current_stream())
    return store


# ---- one pass ---------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    c, op, store = s["case"], s["case"]["op"], s["store"]
    if op == "logprobs":
        return store.token_logprobs(s["z"], s["y"])
    if op == "preference":
        r = store.preference_loss(s["z"], s["y"], s["starts"], s["ref"], beta=BETA,
                                  label_smoothing=c["smoothing"])
        return {"loss": r.loss, "margins": r.margins, "logps": r.logps, "grad": r.grad}
    if op == "policy":
        r = store.policy_loss(s["z"], s["y"], s["old"], s["adv"], s["ref"],
                              clip=(CLIP_LOW, CLIP_HIGH), kl_coef=c["kl"])
        return {"loss": r.loss, "kl": r.kl, "logps": r.logps, "grad": r.grad}
    if op == "checkpoint":
        kept = store.checkpoint8(s["x"], fmt=c["fmt"])
        return store.restore8(kept, dtype=s["x"].dtype)
    if op == "gelu":
        y, kept = store.gelu_checkpoint8(s["x"], fmt=c["fmt"], approximate=c["approximate"])
        dx = store.gelu_backward8(kept, s["dy"], approximate=c["approximate"])
        return {"y": y, "dx": dx}
    import ttperf
    kept = store.checkpoint8(s["x"], fmt=c["fmt"])
    store.zero_grad(set_to_none=True, fill=False)
    store.accumulate_linear_grad8(0, kept, s["dy"], bias=1, transposed=c["transposed"])
    if "views" not in s:  # the buffer's torch views, made once
        s["views"] = {"dw": store.tensors[0].torch_view(ttperf.BUF_GRAD),
                      "db": store.tensors[1].torch_view(ttperf.BUF_GRAD)}
    return s["views"]


def _run_plain(s):
    c, op = s["case"], s["case"]["op"]
    if op == "logprobs":
        return _plain_logps(s["z"], s["y"])[0]
    if op == "preference":
        return _plain_preference(s, c)
    if op == "policy":
        return _plain_policy(s, c)
    x = _plain_kept(s["x"], c["fmt"])
    if op == "checkpoint":
        return x.to(s["x"].dtype)
    dy = s["dy"].float()
    if op == "gelu":
        y, _ = _plain_gelu(s["x"].float(), c["approximate"])
        _, slope = _plain_gelu(x, c["approximate"])
        return {"y": y.to(s["x"].dtype), "dx": (dy * slope).to(s["x"].dtype)}
    dw = torch.mm(dy.t(), x) if c["transposed"] else torch.mm(x.t(), dy)
    return {"dw": dw.to(s["x"].dtype), "db": dy.sum(0).to(s["x"].dtype)}


def _plain_logps(z, y):
    """Log-probabilities of the tokens (0 on masked rows), the exponentials with their sums, and
    the row mask."""
    z, live = z.float(), y >= 0
    top = z.max(1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    at = z.gather(1, y.clamp(min=0)[:, None])
    logp = (at - top - torch.log(total))[:, 0]
    return torch.where(live, logp, 0.0), (e, total), live


def _plain_grad(p, y, live, coef, dtype):
    """coef (1[v = y] - p) on the rows that count, 0 on the others."""
    e, total = p
    g = e.mul_(-coef[:, None] / total)
    rows = torch.arange(len(y), device=y.device)
    g[rows, y.clamp(min=0)] += coef
    return torch.where(live[:, None], g, 0.0).to(dtype)


def _plain_preference(s, c):
    logp, p, live = _plain_logps(s["z"], s["y"])
    pairs, eps = c["pairs"], c["smoothing"]
    seq = torch.bucketize(torch.arange(c["rows"], device="cuda"), s["starts"][1:], right=True)
    member = seq[None, :] == torch.arange(2 * pairs, device="cuda")[:, None]
    ratio = torch.where(member & live, logp - s["ref"], 0.0).sum(1)
    h = BETA * (ratio[:pairs] - ratio[pairs:])
    log_sig = torch.minimum(h, torch.zeros_like(h)) - torch.log1p(torch.exp(-h.abs()))
    loss = (-(1 - eps) * log_sig - eps * (log_sig - h)).mean()
    sig = 1 / (1 + torch.exp(-h))
    dh = (-(1 - eps) * (1 - sig) + eps * sig) * (BETA / pairs)
    coef = torch.cat([dh, -dh])[seq]
    return {"loss": loss, "margins": h, "logps": logp,
            "grad": _plain_grad(p, s["y"], live, coef, s["z"].dtype)}


def _plain_policy(s, c):
    logp, p, live = _plain_logps(s["z"], s["y"])
    count = live.sum().clamp(min=1)
    r = torch.exp(logp - s["old"])
    plain, clipped = r * s["adv"], r.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * s["adv"]
    loss = -torch.minimum(plain, clipped)
    coef = torch.where(plain <= clipped, -plain, 0.0)
    kl = torch.zeros_like(loss)
    if s["ref"] is not None:
        d = s["ref"] - logp
        kl = torch.expm1(d) - d
        coef = coef - c["kl"] * torch.expm1(d)
    loss = torch.where(live, loss + c["kl"] * kl, 0.0).sum() / count
    return {"loss": loss, "kl": torch.where(live, kl, 0.0).sum() / count, "logps": logp,
            "grad": _plain_grad(p, s["y"], live, coef / count, s["z"].dtype)}


def _plain_kept(x, fmt):
    """The values an 8-bit checkpoint stands for: per block of 32 columns the least power of two
    that holds the largest value in 8 bits, the rest rounded to its grid (ties to even)."""
    rows, cols = x.shape
    full = -(-cols // BLOCK) * BLOCK
    b = torch.nn.functional.pad(x.float(), (0, full - cols)).view(rows, -1, BLOCK)
    most = 127.0 if fmt == "int8" else 448.0
    mant, power = torch.frexp(b.abs().amax(2, keepdim=True))
    top_mant, top_power = math.frexp(most)
    e = power - top_power + (mant > top_mant)
    scale = torch.ldexp(torch.ones_like(mant), e)
    q = b / scale
    q = q.round() if fmt == "int8" else q.to(torch.float8_e4m3fn).float()
    return (q * scale).view(rows, full)[:, :cols]


def _plain_gelu(x, approximate):
    """GELU and its derivative."""
    if approximate == "tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (x + 0.044715 * x * x * x))
        inner = k * (1 + 3 * 0.044715 * x * x)
        return 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * inner
    phi = 0.5 * (1 + torch.erf(x / math.sqrt(2)))
    return x * phi, phi + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)


# ---- the definitions in 64 bits ---------------------------------------------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)
    op = c["op"]
    if op in ("logprobs", "preference", "policy"):
        return _exact_loss(c, s)
    x = s["x"].double()
    kept = torch.empty_like(x)
    most = 127.0 if c["fmt"] == "int8" else 448.0
    for a in range(0, c["cols"], BLOCK):  # block by block of columns
        b = x[:, a:a + BLOCK]
        top = b.abs().amax(1, keepdim=True)
        scale = torch.exp2(torch.ceil(torch.log2(top / most)))
        scale = torch.where(scale * most < top, scale * 2, scale)
        scale = torch.where(scale / 2 * most >= top, scale / 2, scale)
        scale = torch.where(top > 0, scale, 1.0)
        v = b / scale
        if c["fmt"] == "int8":
            v = torch.round(v)
        else:  # 3 bits behind the leading one, exponents from -6 on
            step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
            v = torch.round(v / step) * step
        kept[:, a:a + BLOCK] = v * scale
    if op == "checkpoint":
        return kept
    dy = s["dy"].double()
    if op == "linear":
        dw = kept.t() @ dy
        return {"dw": dw.t().contiguous() if c["transposed"] else dw, "db": dy.sum(0)}
    if c["approximate"] == "tanh":
        def gelu(v):
            a = math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
            half = torch.sigmoid(2 * a)
            slope = math.sqrt(2 / math.pi) * (1 + 0.134145 * v ** 2)
            return v * half, half + 2 * v * half * torch.sigmoid(-2 * a) * slope
    else:
        def gelu(v):
            half = torch.special.ndtr(v)
            return v * half, half + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    return {"y": gelu(x)[0], "dx": dy * gelu(kept)[1]}


def _exact_loss(c, s):
    z, y, rows = s["z"], s["y"], c["rows"]
    live = y >= 0
    lse = torch.cat([torch.logsumexp(p.double(), 1) for p in z.split(1024)])
    logp = z.gather(1, y.clamp(min=0)[:, None])[:, 0].double() - lse
    logp = logp * live
    if c["op"] == "logprobs":
        return logp
    out = {"logps": logp}
    coef = torch.zeros(rows, dtype=torch.float64, device="cuda")
    if c["op"] == "preference":
        at, pairs, eps = s["starts"].tolist(), c["pairs"], c["smoothing"]
        d = (logp - s["ref"].double()) * live
        total = torch.stack([d[a:b].sum() for a, b in zip(at, at[1:])])
        h = BETA * (total[:pairs] - total[pairs:])
        soft = torch.nn.functional.softplus
        out["loss"] = ((1 - eps) * soft(-h) + eps * soft(h)).mean()
        out["margins"] = h
        dh = BETA * (torch.sigmoid(h) - (1 - eps)) / pairs
        for k, (a, b) in enumerate(zip(at, at[1:])):
            coef[a:b] = dh[k] if k < pairs else -dh[k - pairs]
    else:
        n = max(int(live.sum()), 1)
        adv = s["adv"].double()
        ratio = torch.exp(logp - s["old"].double())
        low = torch.where(adv >= 0, ratio < 1 + CLIP_HIGH, ratio > 1 - CLIP_LOW)
        held = torch.where(adv >= 0, ratio.clamp(max=1 + CLIP_HIGH), ratio.clamp(min=1 - CLIP_LOW))
        loss, kl = -held * adv, torch.zeros_like(adv)
        coef = -ratio * adv * low
        if s["ref"] is not None:
            gap = s["ref"].double() - logp
            kl = torch.exp(gap) - gap - 1
            coef = coef + c["kl"] * (1 - torch.exp(gap))
        out["loss"] = ((loss + c["kl"] * kl) * live).sum() / n
        out["kl"] = (kl * live).sum() / n
        coef = coef / n
    coef = coef * live
    grad = torch.empty(z.shape, dtype=torch.float64, device="cuda")
    for a in range(0, rows, 1024):
        b = slice(a, a + 1024)
        grad[b] = torch.exp(z[b].double() - lse[b, None]) * -coef[b, None]
    grad[torch.arange(rows, device="cuda"), y.clamp(min=0)] += coef
    out["grad"] = grad
    return {k: out[k] for k in (("loss", "margins", "logps", "grad")
                                if c["op"] == "preference" else ("loss", "kl", "logps", "grad"))}


# ---- what a pass cannot do without ------------------------------------------------------------
def work(case):
    """Bytes: each input read once, each output written once; a checkpoint is written by the
    forward and read by the backward.  Operations: about 4 per logit for a sum of exponentials
    and 4 more for its gradient; 8 per packed value, 20 per GELU."""
    c, op, rows = case, case["op"], case["rows"]
    size = 2 if c["dtype"] == "bf16" else 4
    if op in ("logprobs", "preference", "policy"):
        logits = rows * c["vocab"]
        vectors = {"logprobs": 12, "preference": 16, "policy": 20 + (4 if c.get("kl") else 0)}[op]
        passes = 1 if op == "logprobs" else 2
        return {"bytes": passes * logits * size + rows * vectors, "flops": 4 * passes * logits}
    n = rows * c["cols"]
    kept = 2 * (n + rows * -(-c["cols"] // BLOCK))  # written, and read again
    if op == "checkpoint":
        return {"bytes": 2 * n * size + kept, "flops": 16 * n}
    if op == "gelu":
        return {"bytes": 4 * n * size + kept, "flops": 48 * n}
    m = c["outs"]
    return {"bytes": (n + rows * m + c["cols"] * m + m) * size + kept,
            "flops": 2 * n * m + 8 * n + rows * m}
