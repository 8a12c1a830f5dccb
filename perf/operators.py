"""The timed work of the operators that a program needs beside the quantized products to serve many sequences together.

One step of such a program takes the projections of each sequence's new tokens (one for a sequence that is being answered, a chunk
of a prompt for one that is being read), gives queries and keys their rotary positions, puts the new keys and values into
the pages of a cache, attends over the pages, and at the end draws a token from each sequence's logits.  The kinds of cases:

  rope    rotary positions of a [tokens x heads x dim] tensor
  store   the same for the rows of a fused QKV projection, with the optional norm of each head; keys and values go into the pages
  attend  attention of the new tokens over the paged cache, their own keys and values (stored before) among it
  sample  temperature, top-k, top-p, min-p and the draw, from given random numbers

Where `own` is false the operators are computed by elementary torch operations in 32 bits (angles and sampling in 64), else by the
framework's entry points.  A case is a dict of plain values whose `kind` names the operator.
"""
import math
import random

import numpy as np
import torch

own = False

ELEMENT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # two dozen sequences at one token each, through the query heads of an 8B model: the smallest call, latency counts
        {"name": "rope_decode", "kind": "rope", "tokens": 24, "heads": 32, "dim": 128, "rotated": 128, "mode": 2, "base": 500000.0,
         "scaling": "factors", "far": 8000},
        # a long prompt with half of each head rotated in adjacent pairs, its angles scaled for a context beyond the trained one
        {"name": "rope_prompt", "kind": "rope", "tokens": 2048, "heads": 32, "dim": 128, "rotated": 64, "mode": 0, "base": 10000.0,
         "scaling": "yarn", "far": 100000},
        # the new token of two dozen sequences into 16-token pages of halfs, heads normed first
        {"name": "store_decode", "kind": "store", "seqs": 24, "new": 1, "context": 900, "ragged": True, "layout": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotated": 128, "mode": 2, "base": 1000000.0, "scaling": "none", "norm": True, "type": "f16",
         "page": 16, "order": "token"},
        # the prompts of three requests read together (2048 tokens at most each)
        {"name": "store_prompt", "kind": "store", "seqs": 3, "new": 2048, "context": 4001, "ragged": True, "layout": 2, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotated": 128, "mode": 2, "base": 500000.0, "scaling": "linear", "norm": False, "type": "bf16",
         "page": 64, "order": "head"},
        # one sequence answered at a context of 4001: few rows, the latency of the whole call counts
        {"name": "attend_decode", "kind": "attend", "seqs": 1, "new": 1, "context": 4001, "ragged": False, "layout": 3, "heads": 32,
         "kv_heads": 8, "dim": 128, "type": "f16", "page": 16, "order": "token", "window": 0, "sinks": False},
        # 32 sequences of very different lengths answered together: the bytes of the cache count
        {"name": "attend_batch", "kind": "attend", "seqs": 32, "new": 1, "context": 8192, "ragged": True, "layout": 4, "heads": 32,
         "kv_heads": 8, "dim": 128, "type": "f16", "page": 16, "order": "token", "window": 0, "sinks": False},
        # a prompt chunk of 512 tokens behind a prefix that is in the cache
        {"name": "attend_chunk", "kind": "attend", "seqs": 1, "new": 512, "context": 4096, "ragged": False, "layout": 5, "heads": 32,
         "kv_heads": 8, "dim": 128, "type": "f16", "page": 64, "order": "head", "window": 0, "sinks": False},
        # the last chunk of a long prompt
        {"name": "attend_long", "kind": "attend", "seqs": 1, "new": 2048, "context": 16384, "ragged": False, "layout": 6, "heads": 32,
         "kv_heads": 8, "dim": 128, "type": "f16", "page": 64, "order": "token", "window": 0, "sinks": False},
        # prompts and answers in one step of a model with a sliding window and a learned logit per head that takes part in the
        # softmax only
        {"name": "attend_window", "kind": "attend", "seqs": 7, "new": 700, "context": 6000, "ragged": True, "layout": 7, "heads": 64,
         "kv_heads": 8, "dim": 64, "type": "bf16", "page": 24, "order": "token", "window": 128, "sinks": True},
        # a ragged chunk of a prompt over the one fp32 cache per layer that the whole-layer decode goes on with
        {"name": "attend_dense", "kind": "attend", "seqs": 1, "new": 333, "context": 2049, "ragged": False, "layout": 8, "heads": 32,
         "kv_heads": 8, "dim": 128, "type": "f32", "page": 4096, "order": "head", "window": 0, "sinks": False},
        # one answer's next token
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": 128256, "mix": 0},
        # next tokens of 64 requests, each with settings of its own
        {"name": "sample_batch", "kind": "sample", "rows": 64, "vocab": 128256, "mix": 1},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))




def draw(rng):
    kind = rng.choice(["rope", "store", "store", "attend", "attend", "attend", "attend", "attend", "sample", "sample"])
    if kind == "sample":
        vocab = _log_int(rng, 1000, 262144)
        return {"kind": kind, "rows": _log_int(rng, 1, max(1, min(256, 64 * 128256 // vocab))), "vocab": vocab, "mix": rng.randint(0, 4)}
    dim = rng.choice([64, 64, 80, 96, 112, 128, 128, 128, 192, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 12])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
    turn = {"dim": dim, "rotated": rng.choice([dim, dim, dim // 2, dim // 4 * 2]), "mode": rng.choice([0, 2]),
            "base": rng.choice([10000.0, 500000.0, 1000000.0]), "scaling": rng.choice(["none", "linear", "yarn", "factors"])}
    if kind == "rope":
        return {"kind": kind, "tokens": _log_int(rng, 1, 2048), "heads": rng.randint(1, 32), **turn, "far": _log_int(rng, 100, 1000000)}
    cache = {"heads": heads, "kv_heads": kv_heads, "type": rng.choice(["f16", "f16", "bf16", "f32"]), "page": rng.choice([1, 5, 16, 16, 24, 32, 64, 100, 256]),
             "order": rng.choice(["token", "head"]), "ragged": rng.random() < 0.7, "layout": rng.randint(10, 10 ** 6)}
    if kind == "store":
        seqs = _log_int(rng, 1, 64)
        new = _log_int(rng, 1, max(1, 2048 // seqs))
        return {"kind": kind, "seqs": seqs, "new": new, "context": max(new, _log_int(rng, 1, 1024)), **cache, **turn, "norm": rng.random() < 0.5}
    if rng.random() < 0.5:                                            # answers: one token (or a few speculated ones) a sequence
        seqs, new = _log_int(rng, 1, 64), rng.choice([1, 1, 1, 2, 3, 5])
        context = _log_int(rng, max(new, 16), min(32768, 32 * 8192 * 8 // (seqs * kv_heads)))
    else:                                                             # prompts
        seqs, new = _log_int(rng, 1, 8), _log_int(rng, 2, 2048)
        context = _log_int(rng, new, max(new + 1, min(16384, 16384 * 2048 * 32 // (seqs * heads * new * (1 + dim // 129)))))
    return {"kind": kind, "seqs": seqs, "new": new, "context": context, **cache, "dim": dim,
            "window": rng.choice([0, 0, 0, _log_int(rng, 1, 4096)]), "sinks": rng.random() < 0.3}


class _State:
    pass


def _normal(shape, generator, sigma=1.0, mean=0.0):
    return torch.randn(shape, generator=generator, device="cuda", dtype=torch.float32) * sigma + mean


def _uniform(shape, generator, low=0.0, high=1.0):
    return torch.rand(shape, generator=generator, device="cuda", dtype=torch.float32) * (high - low) + low


def _lengths(case):
    """(new tokens, tokens in the cache with them) of each sequence; the case's own, whatever the seed"""
    r = random.Random(case["layout"])
    news, contexts = [], []
    for i in range(case["seqs"]):
        n = _log_int(r, 1, case["new"]) if case["ragged"] and i else case["new"]
        news.append(n)
        contexts.append(r.randint(n, max(n, case["context"])) if case["ragged"] and i else max(n, case["context"]))
    return news, contexts


def _sequences(s, case, g):
    """row_starts, context_lens and the page table, and a cache of as many pages as the sequences have"""
    news, contexts = _lengths(case)
    page = case["page"]
    s.row_starts = torch.tensor([0] + list(np.cumsum(news)), dtype=torch.int32, device="cuda")
    s.context_lens = torch.tensor(contexts, dtype=torch.int32, device="cuda")
    s.tokens, s.most_new, s.most_context = sum(news), max(news), max(contexts)
    counts = [-(-c // page) for c in contexts]
    s.pages = sum(counts)
    order = torch.randperm(s.pages, generator=g, device="cuda").to(torch.int32).cpu().numpy()
    table = np.full((case["seqs"], max(counts)), -1, dtype=np.int32)      # (entries behind a sequence's last page are not read)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    s.page_table = torch.from_numpy(table).cuda()
    s.k, s.v = (_pages(case, s.pages, g) for _ in range(2))


def _pages(case, count, g):
    """[pages, tokens of a page, heads, dim], the heads before or behind the tokens in memory"""
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    shape = (count, page, heads, dim) if case["order"] == "token" else (count, heads, page, dim)
    t = torch.empty(shape, dtype=ELEMENT[case["type"]], device="cuda")
    t.normal_(generator=g)
    return t if case["order"] == "token" else t.transpose(1, 2)


def _turn(s, case, g):
    s.freq_factors = _uniform((case["rotated"] // 2,), g, 1.0, 8.0) if case["scaling"] == "factors" else None
    s.scaling = {"none": {}, "factors": {}, "linear": {"freq_scale": 0.25},
                 "yarn": {"freq_scale": 0.0625, "ext_factor": 1.0, "attn_factor": 1.0, "beta_fast": 32.0, "beta_slow": 1.0,
                          "original_context": 8192}}[case["scaling"]]


def prepare(case, seed):
    s = _State()
    s.case = case
    s.kind = case["kind"]
    s.handle = None
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if s.kind == "rope":
        s.x = _normal((case["tokens"], case["heads"], case["dim"]), g)
        s.positions = torch.randint(0, case["far"], (case["tokens"],), generator=g, device="cuda").to(torch.int32)
        s.result = torch.empty_like(s.x)
        _turn(s, case, g)
    elif s.kind == "store":
        _sequences(s, case, g)
        s.qkv = _normal((s.tokens, (case["heads"] + 2 * case["kv_heads"]) * case["dim"]), g)
        s.q_norm = _normal((case["dim"],), g, 0.1, 1.0) if case["norm"] else None
        s.k_norm = _normal((case["dim"],), g, 0.1, 1.0) if case["norm"] else None
        s.query = torch.empty((s.tokens, case["heads"] * case["dim"]), dtype=torch.float32, device="cuda")
        _turn(s, case, g)
    elif s.kind == "attend":
        _sequences(s, case, g)
        s.query = _normal((s.tokens, case["heads"] * case["dim"]), g, 2.0)
        s.sinks = _normal((case["heads"],), g) if case["sinks"] else None
        s.result = torch.empty_like(s.query)
    else:
        rows, vocab = case["rows"], case["vocab"]
        s.logits = _normal((rows, vocab), g, 2.0)
        # what the model finds likely stands out of the rest, as it does where a model has learned something
        s.logits.scatter_add_(1, torch.randint(0, vocab, (rows, 60), generator=g, device="cuda"), _uniform((rows, 60), g, 0.0, 14.0))
        s.uniforms = torch.rand((rows,), generator=g, device="cuda", dtype=torch.float32)
        temperature, top_k, top_p, min_p = _settings(case)
        s.temperature, s.top_p, s.min_p = (torch.tensor(v, dtype=torch.float32, device="cuda") for v in (temperature, top_p, min_p))
        s.top_k = torch.tensor(top_k, dtype=torch.int32, device="cuda")
        s.tokens = torch.empty((rows,), dtype=torch.int32, device="cuda")
        s.probabilities = torch.empty((rows,), dtype=torch.float32, device="cuda")
    return s


def _settings(case):
    """temperature, top_k, top_p and min_p of each row: what requests commonly ask for (mix 0: top-k and top-p, 1: each row its own,
    2: none, 3: top-p alone, 4: greedy and min-p rows in turn)"""
    r = random.Random(case["mix"])
    rows = []
    for i in range(case["rows"]):
        mix = case["mix"] if case["mix"] != 1 else r.choice([0, 0, 2, 3, 4])
        rows.append({0: (0.8, 40, 0.95, 0.0), 2: (1.0, 0, 1.0, 0.0), 3: (0.7, 0, 0.9, 0.0),
                     4: (0.0, 0, 1.0, 0.0) if i % 2 else (1.2, 0, 1.0, 0.05)}[mix])
    return tuple(list(v) for v in zip(*rows))


# ---- the plain forms -------------------------------------------------------------------------------------------------------------


def _angles(case, scaling, freq_factors, positions):
    """cos and sin [tokens, rotated / 2] of the angles, in 64 bits up to the last step"""
    n, base = case["rotated"], case["base"]
    pair = torch.arange(n // 2, dtype=torch.float64, device=positions.device)
    frequency = torch.pow(torch.tensor(base, dtype=torch.float64, device=positions.device), -2.0 * pair / n)
    if freq_factors is not None:
        frequency = frequency / freq_factors.double()
    freq_scale, ext = scaling.get("freq_scale", 1.0), scaling.get("ext_factor", 0.0)
    size = scaling.get("attn_factor", 1.0)
    if ext:
        border = [n * math.log(scaling["original_context"] / (b * 2 * math.pi)) / (2 * math.log(base)) for b in (scaling["beta_fast"], scaling["beta_slow"])]
        low, high = max(0.0, math.floor(border[0])), min(n - 1.0, math.ceil(border[1]))
        kept = (1.0 - ((pair - low) / max(0.001, high - low)).clamp(0.0, 1.0)) * ext
        frequency = frequency * (freq_scale * (1.0 - kept) + kept)
        size *= 1.0 + 0.1 * math.log(1.0 / freq_scale)
    else:
        frequency = frequency * freq_scale
    theta = positions.double()[:, None] * frequency[None, :]
    return (torch.cos(theta) * size).float(), (torch.sin(theta) * size).float()


def _rotated(x, case, cos, sin):
    """x [tokens, heads, dim] with its first `rotated` dimensions turned"""
    n = case["rotated"]
    first, rest = x[..., :n], x[..., n:]
    c, s = cos[:, None, :], sin[:, None, :]
    if case["mode"] == 2:
        a, b = first[..., :n // 2], first[..., n // 2:]
        turned = torch.cat([a * c - b * s, a * s + b * c], dim=-1)
    else:
        a, b = first[..., 0::2], first[..., 1::2]
        turned = torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2)
    return torch.cat([turned, rest], dim=-1)


def _places(s):
    """sequence, position in it and place among its new tokens of each row"""
    rows = torch.arange(s.tokens, device="cuda")
    seq = torch.searchsorted(s.row_starts.long(), rows, right=True) - 1
    starts = s.row_starts.long()
    new = starts[seq + 1] - starts[seq]
    within = rows - starts[seq]
    return seq, s.context_lens.long()[seq] - new + within, within


def _plain_rope(s):
    cos, sin = _angles(s.case, s.scaling, s.freq_factors, s.positions)
    return _rotated(s.x, s.case, cos, sin)


def _head_norm(x, weight):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight if weight is not None else x


def _plain_store(s):
    c = s.case
    heads, kv, dim = c["heads"], c["kv_heads"], c["dim"]
    seq, position, _ = _places(s)
    cos, sin = _angles(c, s.scaling, s.freq_factors, position)
    x = s.qkv.view(s.tokens, heads + 2 * kv, dim)
    q = _rotated(_head_norm(x[:, :heads], s.q_norm), c, cos, sin)
    k = _rotated(_head_norm(x[:, heads:heads + kv], s.k_norm), c, cos, sin)
    page = s.page_table.long()[seq, position // c["page"]]
    s.k[page, position % c["page"]] = k.to(s.k.dtype)
    s.v[page, position % c["page"]] = x[:, heads + kv:].to(s.v.dtype)
    return {"query": q.reshape(s.tokens, heads * dim), "k": s.k, "v": s.v}


def _plain_attend(s):
    c = s.case
    seqs, heads, kv, dim = c["seqs"], c["heads"], c["kv_heads"], c["dim"]
    group, most = heads // kv, s.most_new
    starts, contexts = s.row_starts.long(), s.context_lens.long()
    # the sequences' pages as [seqs, kv heads, positions, dim], the rows of the new tokens as [seqs, kv heads, group x new, dim]
    j = torch.arange(s.most_context, device="cuda")
    page = s.page_table.long()[:, j // c["page"]].clamp(min=0)
    k, v = (t[page, j % c["page"]].float().permute(0, 2, 1, 3) for t in (s.k, s.v))
    i = torch.arange(most, device="cuda")
    new = starts[1:] - starts[:-1]
    row = (starts[:-1, None] + i).clamp(max=s.tokens - 1)
    q = s.query.view(s.tokens, kv, group, dim)[row].permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * most, dim)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).view(seqs, kv, group, most, -1) * (1.0 / math.sqrt(dim))
    position = (contexts - new)[:, None] + i
    seen = j[None, None, :] <= position[:, :, None]
    if c["window"]:
        seen &= j[None, None, :] > position[:, :, None] - c["window"]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    if s.sinks is not None:
        top = torch.maximum(top, s.sinks.view(1, kv, group, 1, 1))
    weights = torch.exp(scores.sub_(top))
    total = weights.sum(-1, keepdim=True)
    if s.sinks is not None:
        total = total + torch.exp(s.sinks.view(1, kv, group, 1, 1) - top)
    out = torch.matmul(weights.view(seqs, kv, group * most, -1), v.contiguous()).view(seqs, kv, group, most, dim) / total
    seq, _, within = _places(s)
    return out.permute(0, 3, 1, 2, 4)[seq, within].reshape(s.tokens, heads * dim)


def _plain_sample(s):
    rows, vocab = s.logits.shape
    logits = s.logits.double()
    ranked, order = torch.sort(logits, dim=1, descending=True, stable=True)      # ties: the lowest index first
    temperature = s.temperature.double()[:, None]
    greedy = ~(temperature > 0)
    weight = torch.exp((ranked - ranked[:, :1]) / torch.where(greedy, 1.0, temperature))
    rank = torch.arange(vocab, device="cuda")[None, :]
    weight = torch.where((s.top_k[:, None] <= 0) | (rank < s.top_k[:, None]), weight, 0.0)
    before = torch.cumsum(weight, 1) - weight
    p = s.top_p.double()[:, None]
    kept = (p >= 1) | (before < p * weight.sum(1, keepdim=True))
    kept &= weight >= s.min_p.double()[:, None]
    kept &= ~greedy
    kept[:, 0] = True                                                            # the likeliest always stays
    weight = torch.zeros_like(weight).scatter_(1, order, torch.where(kept, weight, 0.0))
    cumulated = torch.cumsum(weight, 1)
    total = cumulated[:, -1:]
    token = (cumulated <= s.uniforms.double()[:, None] * total).sum(1, keepdim=True)
    return {"tokens": token[:, 0].to(torch.int32), "probabilities": (weight.gather(1, token) / total)[:, 0].float()}


# ---- the calls -------------------------------------------------------------------------------------------------------------------


def _handle(s):
    """what a program makes once and keeps: the description of the rotation, and of the cache with its page table"""
    if s.handle is None:
        from tensorsharp_amd import PagedKVCache, RotaryPositions
        c = s.case
        rope = RotaryPositions(c["rotated"], mode=c["mode"], base=c["base"], freq_factors=s.freq_factors, **s.scaling) if s.kind != "attend" else None
        s.handle = (rope, PagedKVCache(s.k, s.v, s.page_table) if s.kind != "rope" else None)
    return s.handle


def run(s):
    if own:
        from tensorsharp_amd import HipBasicOps
        if s.kind == "rope":
            HipBasicOps.RoPE(s.result, s.x, s.positions, _handle(s)[0])
            return s.result
        if s.kind == "store":
            rope, cache = _handle(s)
            HipBasicOps.RoPEStorePaged(s.query, s.qkv, cache, s.row_starts, s.context_lens, rope, s.q_norm, s.k_norm, 1e-6)
            return {"query": s.query, "k": s.k, "v": s.v}
        if s.kind == "attend":
            HipBasicOps.PagedAttention(s.result, s.query, _handle(s)[1], s.row_starts, s.context_lens, 1.0 / math.sqrt(s.case["dim"]),
                                       window=s.case["window"], sinks=s.sinks)
            return s.result
        HipBasicOps.SampleTokens(s.tokens, s.logits, s.uniforms, s.temperature, s.top_k, s.top_p, s.min_p, s.probabilities)
        return {"tokens": s.tokens, "probabilities": s.probabilities}
    return {"rope": _plain_rope, "store": _plain_store, "attend": _plain_attend, "sample": _plain_sample}[s.kind](s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------------


def work(case):
    if case["kind"] == "rope":
        values = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 8 * values + 4 * case["tokens"], "flops": 3 * case["tokens"] * case["heads"] * case["rotated"]}
    if case["kind"] == "sample":
        return {"bytes": 4 * case["rows"] * (case["vocab"] + 7), "flops": 4 * case["rows"] * case["vocab"]}
    news, contexts = _lengths(case)
    tokens, size = sum(news), {"f32": 4, "f16": 2, "bf16": 2}[case["type"]]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "store":
        return {"bytes": 4 * tokens * (2 * heads + 2 * kv) * dim + 2 * size * tokens * kv * dim,
                "flops": 3 * tokens * (heads + kv) * case["rotated"]}
    window = case["window"] or 1 << 40
    pairs = keys = 0
    for n, ctx in zip(news, contexts):
        first = ctx - n                                               # position of the first new token: it sees min(first + 1, window) keys
        full = min(n, max(0, window - first - 1))                     # tokens that the window does not cut
        pairs += full * first + full * (full + 1) // 2 + (n - full) * min(window, ctx)
        keys += min(ctx, window + n - 1)
    return {"bytes": 8 * tokens * heads * dim + 2 * size * keys * kv * dim, "flops": 4 * pairs * heads * dim}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------


def _exact_turn(x, case, s, positions):
    """float64 [tokens, heads, dim] -> the same, turned as complex numbers"""
    n = case["rotated"]
    i = np.arange(n // 2, dtype=np.float64)
    w = case["base"] ** (-2.0 * i / n)
    if s.freq_factors is not None:
        w = w / s.freq_factors.cpu().numpy().astype(np.float64)
    y, size = s.scaling, 1.0
    if y.get("ext_factor"):
        edge = lambda beta: n * np.log(y["original_context"] / (2.0 * np.pi * beta)) / (2.0 * np.log(case["base"]))  # noqa: E731
        low, high = max(np.floor(edge(y["beta_fast"])), 0.0), min(np.ceil(edge(y["beta_slow"])), n - 1.0)
        share = (1.0 - np.minimum(1.0, np.maximum(0.0, (i - low) / max(high - low, 1e-3)))) * y["ext_factor"]
        w = w * y["freq_scale"] * (1.0 - share) + w * share
        size = y["attn_factor"] * (1.0 - 0.1 * np.log(y["freq_scale"]))
    elif y:
        w = w * y["freq_scale"]
    turn = size * torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                              positions.double()[:, None] * torch.from_numpy(w).to(x.device)[None])[:, None, :]
    out = x.clone()
    at = (slice(0, n // 2), slice(n // 2, n)) if case["mode"] == 2 else (slice(0, n, 2), slice(1, n, 2))
    z = torch.complex(x[..., at[0]].contiguous(), x[..., at[1]].contiguous()) * turn
    out[..., at[0]], out[..., at[1]] = z.real, z.imag
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "rope":
        return _exact_turn(s.x.double(), case, s, s.positions)
    if s.kind == "sample":
        return _exact_sample(s)
    news, contexts = _lengths(case)
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    table = s.page_table.long()
    if s.kind == "store":
        x = s.qkv.double().view(s.tokens, -1, dim)
        position = torch.cat([torch.arange(c - n, c, device="cuda") for n, c in zip(news, contexts)])
        seq = torch.cat([torch.full((n,), b, device="cuda") for b, n in enumerate(news)])
        parts = []
        for at, w in ((slice(0, heads), s.q_norm), (slice(heads, heads + kv), s.k_norm)):
            y = x[:, at]
            if w is not None:
                y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / dim + 1e-6) * w.double()
            parts.append(_exact_turn(y, case, s, position))
        k, v = s.k.double(), s.v.double()
        where = (table[seq, torch.div(position, page, rounding_mode="floor")], torch.remainder(position, page))
        k[where], v[where] = parts[1], x[:, heads + kv:]
        return {"query": parts[0].reshape(s.tokens, heads * dim), "k": k, "v": v}
    out = torch.zeros((s.tokens, heads, dim), dtype=torch.float64, device="cuda")
    row = 0
    for b, (n, ctx) in enumerate(zip(news, contexts)):
        j = torch.arange(ctx, device="cuda")
        at = (table[b, torch.div(j, page, rounding_mode="floor")], torch.remainder(j, page))
        back = torch.arange(ctx - n, ctx, device="cuda")[:, None] - j[None, :]      # how far behind the token a key lies
        hidden = (back < 0) | (back >= case["window"]) if case["window"] else back < 0
        for h in range(heads):
            g = h // (heads // kv)
            q = s.query[row:row + n].view(n, heads, dim)[:, h].double()
            z = (q @ s.k[at][:, g].double().t().contiguous()) / math.sqrt(dim)
            z[hidden] = -math.inf
            if s.sinks is not None:
                z = torch.cat([z, s.sinks[h].double().expand(n, 1)], dim=1)
            z = torch.exp(z - z.max(1, keepdim=True).values)
            out[row:row + n, h] = (z[:, :ctx] @ s.v[at][:, g].double()) / z.sum(1, keepdim=True)
        row += n
    return out.view(s.tokens, heads * dim)


def _exact_sample(s):
    logits = s.logits.cpu().numpy().astype(np.float64)
    settings = [t.cpu().numpy().astype(np.float64) for t in (s.uniforms, s.temperature, s.top_k, s.top_p, s.min_p)]
    tokens, probabilities = [], []
    for x, u, t, k, p, m in zip(logits, *settings):
        if t <= 0:
            tokens.append(int(np.argmax(x)))
            probabilities.append(1.0)
            continue
        ids = np.argsort(-x, kind="stable")
        if k > 0:
            ids = ids[:int(k)]
        w = np.exp((x[ids] - x.max()) / t)
        if p < 1:
            ids = ids[:1 + int(np.searchsorted(np.cumsum(w), p * w.sum()))]
        ids = np.sort(ids[(np.exp((x[ids] - x.max()) / t) >= m) | (x[ids] == x.max())])
        w = np.exp((x[ids] - x.max()) / t)
        i = min(int(np.searchsorted(np.cumsum(w), u * w.sum(), side="right")), len(ids) - 1)
        tokens.append(int(ids[i]))
        probabilities.append(w[i] / w.sum())
    return {"tokens": np.array(tokens, dtype=np.int32), "probabilities": np.array(probabilities)}
