"""The timed work of the operators with which many sequences keep long contexts: a cache in four bits, windows with first tokens that stay
visible, and the life of a cache's pages.

The kinds of cases:

  store      norms, rotary positions and the store of new keys and values into pages, which hold them in four bits (MXFP4: blocks of 32
             along a head, a code of sign, two bits of exponent and one of mantissa each, and a power of two for the block)
  attend     attention of new tokens over such a cache, or over one of 16 or 32 bits whose tokens see a window and the first tokens
  fork       sequences go on from what others have: tables, reference counts, and the copies of pages that are begun
  turnover   sequences that have ended give their pages back, prompts in their place get pages
  compact    the same with the pages in use moved together to the front of the memory
  cold       pages copied into a cache of four bits and back into one of 16 or 32

Where `own` is false the operators are computed by elementary torch operations in 32 bits (angles in 64), else by the framework's entry
points.  A case is a dict of plain values whose `kind` names the operator.  What four bits hold is returned as the values it stands for.
"""
import math
import random

import numpy as np
import torch

own = False

ELEMENT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4.0, "f16": 2.0, "bf16": 2.0, "mx4": 17 / 32}                  # bytes of a value
MAGNITUDE = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)                          # of the codes 0 to 7; 8 to 15: negative


def listed():
    heads = {"heads": 32, "kv_heads": 8, "dim": 128}
    turn = {"rotated": 128, "mode": 2, "base": 500000.0, "scaling": "none"}
    return [
        # the new token of two dozen sequences, heads normed first: the smallest store, latency counts
        {"name": "store_answers", "kind": "store", "seqs": 24, "new": 1, "context": 900, "ragged": True, "layout": 1, **heads, **turn,
         "norm": True, "type": "mx4", "page": 16, "order": "token"},
        # the prompts of three requests read together (2048 tokens at most each)
        {"name": "store_prompts", "kind": "store", "seqs": 3, "new": 2048, "context": 2500, "ragged": True, "layout": 2, **heads, **turn,
         "norm": False, "type": "mx4", "page": 64, "order": "head"},
        # one sequence answered at a context of 4001: the latency of the whole call counts
        {"name": "attend_answer", "kind": "attend", "seqs": 1, "new": 1, "context": 4001, "ragged": False, "layout": 3, **heads, "type": "mx4",
         "page": 16, "order": "token", "window": 0, "first": 0, "sinks": False},
        # 32 long sequences of very different lengths answered together: the bytes of the cache count
        {"name": "attend_answers", "kind": "attend", "seqs": 32, "new": 1, "context": 16384, "ragged": True, "layout": 4, **heads,
         "type": "mx4", "page": 64, "order": "head", "window": 0, "first": 0, "sinks": False},
        # a ragged chunk of a prompt behind a prefix that is in the cache
        {"name": "attend_chunk", "kind": "attend", "seqs": 1, "new": 509, "context": 4096, "ragged": False, "layout": 5, **heads, "type": "mx4",
         "page": 64, "order": "token", "window": 0, "first": 0, "sinks": False},
        # answers that never end: each sees its last 1024 positions and the four that the sequence began with
        {"name": "first_answers", "kind": "attend", "seqs": 24, "new": 1, "context": 16000, "ragged": True, "layout": 6, **heads, "type": "f16",
         "page": 16, "order": "token", "window": 1024, "first": 4, "sinks": False},
        # prompts and answers in one step of a model of small heads with a window and a learned logit per head
        {"name": "first_prompts", "kind": "attend", "seqs": 7, "new": 700, "context": 6000, "ragged": True, "layout": 7, "heads": 64,
         "kv_heads": 8, "dim": 64, "type": "bf16", "page": 24, "order": "token", "window": 128, "first": 5, "sinks": True},
        # a step of beam search: each of four beams of eight requests goes on from one of the four
        {"name": "fork_beams", "kind": "fork", "requests": 8, "each": 4, "context": 2000, "more": 40, "beams": True, "layout": 8, "kv_heads": 8,
         "dim": 128, "type": "f16", "page": 16, "order": "token"},
        # one prompt each of 24 requests answered in eight samples
        {"name": "fork_samples", "kind": "fork", "requests": 24, "each": 8, "context": 12000, "more": 1, "beams": False, "layout": 9, "kv_heads": 8,
         "dim": 128, "type": "bf16", "page": 64, "order": "head"},
        # 256 sequences, a quarter of them ends and prompts take their places: lists alone
        {"name": "turnover", "kind": "turnover", "seqs": 256, "context": 6000, "free": 0.1, "layout": 10, "page": 16},
        # the same of 48 sequences, and their pages are moved to the front of a cache
        {"name": "compact", "kind": "compact", "seqs": 48, "context": 2400, "free": 0.3, "layout": 11, "kv_heads": 8, "dim": 128, "type": "f16",
         "page": 32, "order": "token"},
        # 400 pages of sequences that wait, into four bits and back
        {"name": "cold_pages", "kind": "cold", "moved": 400, "kv_heads": 8, "dim": 128, "type": "bf16", "page": 64, "order": "token"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "attend", "first", "first", "fork", "turnover", "compact", "cold"])
    page = rng.choice([1, 5, 16, 16, 24, 32, 64, 100, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 12])
    order = rng.choice(["token", "head"])
    layout = rng.randint(100, 10 ** 6)
    if kind == "turnover":
        return {"kind": kind, "seqs": _log_int(rng, 1, 500), "context": _log_int(rng, 1, 6000), "free": rng.uniform(0.0, 0.5), "layout": layout, "page": page}
    if kind in ("fork", "compact", "cold"):
        dim = rng.choice([32, 64, 96, 128, 128, 192, 256])
        cache = {"kv_heads": kv_heads, "dim": dim, "type": rng.choice(["f16", "bf16", "f32"]), "page": page, "order": order}
        room = 24 * 12000 * 8 * 128 // (kv_heads * dim)              # tokens that a drawn cache may have
        if kind == "cold":
            return {"kind": kind, "moved": _log_int(rng, 1, max(1, min(400, 400 * 64 * 1024 // (page * kv_heads * dim)))), **cache}
        if kind == "fork":
            requests, each = _log_int(rng, 1, 24), rng.choice([1, 2, 3, 4, 8])
            return {"kind": kind, "requests": requests, "each": each, "context": _log_int(rng, 1, max(1, min(12000, room // (2 * requests)))),
                    "more": rng.randint(1, 100), "beams": rng.random() < 0.5, "layout": layout, **cache}
        seqs = _log_int(rng, 1, 64)
        return {"kind": kind, "seqs": seqs, "context": _log_int(rng, 1, max(1, min(4000, room // (2 * seqs)))), "free": rng.uniform(0.0, 0.5),
                "layout": layout, **cache}
    small = kind == "first" and rng.random() < 0.7                   # (windows with first tokens go over caches of all types)
    dim = rng.choice([16, 64, 80, 96, 112, 128, 128, 192, 256] if small else [32, 64, 64, 96, 128, 128, 128, 160, 192, 256])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
    case = {"heads": heads, "kv_heads": kv_heads, "dim": dim, "type": rng.choice(["f16", "bf16", "f32"]) if small else "mx4", "page": page, "order": order,
            "ragged": rng.random() < 0.7, "layout": layout}
    if kind == "store":
        seqs = _log_int(rng, 1, 64)
        new = _log_int(rng, 1, max(1, 2048 // seqs))
        return {"kind": kind, "seqs": seqs, "new": new, "context": max(new, _log_int(rng, 1, 1024)), **case, "norm": rng.random() < 0.5,
                "rotated": rng.choice([dim, dim, dim // 2, dim // 4 * 2 // 4 * 4]), "mode": rng.choice([0, 2]),
                "base": rng.choice([10000.0, 500000.0, 1000000.0]), "scaling": rng.choice(["none", "linear", "yarn", "factors"])}
    if rng.random() < 0.5:                                            # answers: one token (or a few speculated ones) a sequence
        seqs, new = _log_int(rng, 1, 64), rng.choice([1, 1, 1, 2, 3, 5])
        context = _log_int(rng, max(new, 16), min(32768, 32 * 16384 * 8 // (2 * seqs * kv_heads)))
    else:                                                             # prompts
        seqs, new = _log_int(rng, 1, 8), _log_int(rng, 2, 2048)
        context = _log_int(rng, new, max(new + 1, min(16384, 16384 * 2048 * 32 // (seqs * heads * new * (1 + dim // 129)))))
    window = _log_int(rng, 1, 4096) if kind == "first" else rng.choice([0, 0, 0, _log_int(rng, 1, 4096)])
    return {"kind": "attend", "seqs": seqs, "new": new, "context": context, **case, "window": window,
            "first": rng.choice([1, 4, 4, 16, _log_int(rng, 1, 500)]) if kind == "first" else 0, "sinks": rng.random() < 0.3}


class _State:
    pass


def _normal(shape, generator, sigma=1.0, mean=0.0):
    return torch.randn(shape, generator=generator, device="cuda", dtype=torch.float32) * sigma + mean


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- four bits -------------------------------------------------------------------------------------------------------------------


def _coded(x):
    """float32 [.., dim] -> codes [.., dim / 2] (two a byte, the first in the lower bits) and scales [.., dim / 32]: 127 + the least
    power, -126 at least, of which the block's largest is at most seven"""
    block = x.unflatten(-1, (-1, 32))
    top = block.abs().amax(-1)
    mantissa, power = torch.frexp(top.double() / 7.0)
    power = torch.where(mantissa > 0.5, power, power - 1).clamp(min=-126)
    power = torch.where(top > 0, power, -126)
    scale = torch.where(top < 2.0 ** 127, power + 127, 255).to(torch.uint8)
    y = torch.ldexp(block.abs().double(), -power[..., None].double())
    code = sum(((y >= e) if even else (y > e)).to(torch.uint8)
               for e, even in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)))
    code = (code + 8 * torch.signbit(block).to(torch.uint8)).flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2], scale


def _values(codes, scales):
    """float32 values of codes and scales"""
    table = torch.tensor(MAGNITUDE + tuple(-m for m in MAGNITUDE), dtype=torch.float32, device=codes.device)
    value = table[torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).int()].unflatten(-1, (-1, 32))
    power = torch.where(scales == 255, math.nan, torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127))
    return (value * power[..., None]).flatten(-2)


# ---- states ----------------------------------------------------------------------------------------------------------------------


def _lengths(case):
    """(new tokens, tokens in the cache with them) of each sequence; the case's own, whatever the seed"""
    r = random.Random(case["layout"])
    news, contexts = [], []
    for i in range(case["seqs"]):
        n = _log_int(r, 1, case["new"]) if case["ragged"] and i else case["new"]
        news.append(n)
        contexts.append(r.randint(n, max(n, case["context"])) if case["ragged"] and i else max(n, case["context"]))
    return news, contexts


def _ordered(t, order):
    return t if order == "token" else t.transpose(1, 2).contiguous().transpose(1, 2)


def _pages(case, count, g, kind=None, empty=False):
    """[pages, tokens of a page, heads, dim] of the case's type, the heads before or behind the tokens in memory; in four bits a pair of
    codes and scales"""
    page, heads, dim, kind = case["page"], case["kv_heads"], case["dim"], kind or case["type"]
    if kind != "mx4":
        t = torch.zeros((count, page, heads, dim) if case["order"] == "token" else (count, heads, page, dim), dtype=ELEMENT[kind], device="cuda")
        if not empty:
            t.normal_(generator=g)
        return t if case["order"] == "token" else t.transpose(1, 2)
    codes = torch.zeros((count, page, heads, dim // 2), dtype=torch.uint8, device="cuda")
    scales = torch.zeros((count, page, heads, dim // 32), dtype=torch.uint8, device="cuda")
    at_once = max(1, (1 << 26) // (page * heads * dim))
    for i in range(0, 0 if empty else count, at_once):
        n = min(at_once, count - i)
        codes[i:i + n], scales[i:i + n] = _coded(_normal((n, page, heads, dim), g))
    return _ordered(codes, case["order"]), _ordered(scales, case["order"])


def _sequences(s, case, g):
    """row_starts, context_lens and the page table, and a cache of as many pages as the sequences have"""
    news, contexts = _lengths(case)
    page = case["page"]
    s.row_starts = _ints([0] + list(np.cumsum(news)))
    s.context_lens = _ints(contexts)
    s.tokens, s.most_new, s.most_context = sum(news), max(news), max(contexts)
    counts = [-(-c // page) for c in contexts]
    order = torch.randperm(sum(counts), generator=g, device="cuda").to(torch.int32).cpu().numpy()
    table = np.full((case["seqs"], max(counts)), -1, dtype=np.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    s.page_table = torch.from_numpy(table).cuda()
    s.k, s.v = (_pages(case, sum(counts), g) for _ in range(2))
    # the pages that the new tokens go into, one after the other
    written = np.concatenate([table[i, (c - n) // page:-(-c // page)] for i, (n, c) in enumerate(zip(news, contexts))])
    s.written = _ints(np.stack([written, np.arange(len(written))], axis=1).tolist())


def _pool(s, shares, tokens, page, free, g):
    """A pool of pages: sequence i has tokens[i] tokens, its whole pages among the first shares[i] tokens in common with the sequence
    before it.  table, references and lens, and how many pages there are"""
    counts, rows, at = [-(-t // page) for t in tokens], [], 0
    for i, n in enumerate(counts):
        shared = min(n, shares[i] // page) if i else 0
        rows.append((rows[-1][:shared] if shared else []) + list(range(at, at + n - shared)))
        at += n - shared
    pages = at + int(at * free) + len(tokens) + 1
    ids = torch.randperm(pages, generator=g, device="cuda").cpu().numpy()
    table = np.full((len(tokens), max(counts) + 1), -1, dtype=np.int32)
    for i, r in enumerate(rows):
        table[i, :len(r)] = ids[np.array(r, dtype=np.int64)]
    s.table = torch.from_numpy(table).cuda()
    s.references = torch.from_numpy(np.bincount(table[table >= 0], minlength=pages).astype(np.int32)).cuda()
    s.lens = _ints(tokens)
    s.pages = pages


def _tokens(case):
    """tokens of each sequence of a pool, and how many of them it may share with the one before"""
    r = random.Random(case["layout"])
    if case["kind"] != "fork":
        tokens = [r.randint(max(1, case["context"] // 4), max(1, case["context"])) for _ in range(case["seqs"])]
        return tokens, [0] * len(tokens)
    tokens, shares = [], []
    for _ in range(case["requests"]):
        prompt = r.randint(max(1, case["context"] // 4), max(1, case["context"]))
        tokens += [prompt + case["more"]] * case["each"]
        shares += [0] + [prompt] * (case["each"] - 1)
    return tokens, shares


def prepare(case, seed):
    s = _State()
    s.case, s.kind, s.handles, s.turn = case, case["kind"], None, 0
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if s.kind in ("store", "attend"):
        _sequences(s, case, g)
        if s.kind == "store":
            s.qkv = _normal((s.tokens, (case["heads"] + 2 * case["kv_heads"]) * case["dim"]), g)
            s.q_norm = _normal((case["dim"],), g, 0.1, 1.0) if case["norm"] else None
            s.k_norm = _normal((case["dim"],), g, 0.1, 1.0) if case["norm"] else None
            s.query = torch.empty((s.tokens, case["heads"] * case["dim"]), dtype=torch.float32, device="cuda")
            s.freq_factors = torch.rand((case["rotated"] // 2,), generator=g, device="cuda") * 7.0 + 1.0 if case["scaling"] == "factors" else None
            s.scaling = {"none": {}, "factors": {}, "linear": {"freq_scale": 0.25},
                         "yarn": {"freq_scale": 0.0625, "ext_factor": 1.0, "attn_factor": 1.0, "beta_fast": 32.0, "beta_slow": 1.0,
                                  "original_context": 8192}}[case["scaling"]]
            s.out_k, s.out_v = (_pages(case, len(s.written), g, "bf16", empty=True) for _ in range(2))
        else:
            s.query = _normal((s.tokens, case["heads"] * case["dim"]), g, 2.0)
            s.sinks = _normal((case["heads"],), g) if case["sinks"] else None
            s.result = torch.empty_like(s.query)
    elif s.kind == "cold":
        n = case["moved"]
        s.pages = n + n // 4 + 1
        s.warm = [_pages(case, s.pages, g) for _ in range(2)]
        s.cold = [_pages(case, n, g, "mx4", empty=True) for _ in range(2)]
        s.back = [_pages(case, n, g, empty=True) for _ in range(2)]
        of, to = torch.randperm(s.pages, generator=g, device="cuda")[:n], torch.randperm(n, generator=g, device="cuda")
        s.moves = torch.stack([of, to], dim=1).to(torch.int32).contiguous()
        s.returns = torch.stack([to, torch.arange(n, device="cuda")], dim=1).to(torch.int32).contiguous()
        s.page_table = torch.arange(n, dtype=torch.int32, device="cuda")[None]
    else:
        tokens, shares = _tokens(case)
        _pool(s, shares, tokens, case["page"], case.get("free", 0.1), g)
        s.missing = torch.zeros((1,), dtype=torch.int32, device="cuda")
        if s.kind == "fork":
            each, all_seqs = case["each"], torch.arange(len(tokens), device="cuda")
            request = all_seqs // each
            if case["beams"]:
                children, parents = all_seqs, request * each + torch.randint(0, each, (len(tokens),), generator=g, device="cuda")
            else:
                children = all_seqs[(all_seqs % each != 0)] if each > 1 else all_seqs
                parents = children // each * each
            s.children, s.parents = children.to(torch.int32), parents.to(torch.int32)
            s.moves = torch.empty((len(children), 2), dtype=torch.int32, device="cuda")
        else:
            ends = np.arange(len(tokens))[None, :] % 4 == np.arange(4)[:, None]
            s.ended = _ints(np.where(ends, 0, -1).tolist())
            s.admitted = _ints(np.where(ends, np.array(tokens)[None, :], -1).tolist())
            s.begun = torch.empty((len(tokens), 2), dtype=torch.int32, device="cuda")
            s.moves = torch.empty((s.pages // 2 + 1, 2), dtype=torch.int32, device="cuda")
        if s.kind != "turnover":
            s.k, s.v = (_pages(case, s.pages, g) for _ in range(2))
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------------------------


def _places(s):
    """sequence and position in it of each row"""
    rows = torch.arange(s.tokens, device="cuda")
    starts = s.row_starts.long()
    seq = torch.searchsorted(starts, rows, right=True) - 1
    return seq, s.context_lens.long()[seq] - starts[seq + 1] + rows


def _turned(x, case, scaling, freq_factors, position):
    """x [tokens, heads, dim] with its first `rotated` dimensions turned by angles in 64 bits"""
    n, base = case["rotated"], case["base"]
    pair = torch.arange(n // 2, dtype=torch.float64, device=x.device)
    frequency = torch.pow(torch.tensor(base, dtype=torch.float64, device=x.device), -2.0 * pair / n)
    if freq_factors is not None:
        frequency = frequency / freq_factors.double()
    size = scaling.get("attn_factor", 1.0)
    if scaling.get("ext_factor"):
        border = [n * math.log(scaling["original_context"] / (b * 2 * math.pi)) / (2 * math.log(base)) for b in (scaling["beta_fast"], scaling["beta_slow"])]
        low, high = max(0.0, math.floor(border[0])), min(n - 1.0, math.ceil(border[1]))
        kept = (1.0 - ((pair - low) / max(0.001, high - low)).clamp(0.0, 1.0)) * scaling["ext_factor"]
        frequency = frequency * (scaling["freq_scale"] * (1.0 - kept) + kept)
        size *= 1.0 + 0.1 * math.log(1.0 / scaling["freq_scale"])
    else:
        frequency = frequency * scaling.get("freq_scale", 1.0)
    theta = position.double()[:, None] * frequency[None, :]
    c, s = (torch.cos(theta) * size).float()[:, None, :], (torch.sin(theta) * size).float()[:, None, :]
    first, rest = x[..., :n], x[..., n:]
    if case["mode"] == 2:
        a, b = first[..., :n // 2], first[..., n // 2:]
        out = torch.cat([a * c - b * s, a * s + b * c], dim=-1)
    else:
        a, b = first[..., 0::2], first[..., 1::2]
        out = torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2)
    return torch.cat([out, rest], dim=-1)


def _plain_store(s):
    c = s.case
    heads, kv, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    normed = lambda x, w: x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w  # noqa: E731
    seq, position = _places(s)
    x = s.qkv.view(s.tokens, heads + 2 * kv, dim)
    q = _turned(normed(x[:, :heads], s.q_norm), c, s.scaling, s.freq_factors, position)
    k = _turned(normed(x[:, heads:heads + kv], s.k_norm), c, s.scaling, s.freq_factors, position)
    where = (s.page_table.long()[seq, position // page], position % page)
    out = {"query": q.reshape(s.tokens, heads * dim)}
    pages = s.written[:, 0].long()
    for name, new, cache in (("k", k, s.k), ("v", x[:, heads + kv:], s.v)):
        codes, scales = _coded(new)
        cache[0][where], cache[1][where] = codes, scales
        out[name] = _values(cache[0][pages], cache[1][pages]).bfloat16()
    return out


def _plain_attend(s):
    c = s.case
    seqs, heads, kv, dim = c["seqs"], c["heads"], c["kv_heads"], c["dim"]
    group, most = heads // kv, s.most_new
    starts, contexts = s.row_starts.long(), s.context_lens.long()
    # the sequences' pages as [seqs, kv heads, positions, dim], the rows of the new tokens as [seqs, kv heads, group x new, dim]
    j = torch.arange(s.most_context, device="cuda")
    at = (s.page_table.long()[:, j // c["page"]].clamp(min=0), j % c["page"])
    k, v = ((_values(t[0][at], t[1][at]) if c["type"] == "mx4" else t[at].float()).permute(0, 2, 1, 3) for t in (s.k, s.v))
    i = torch.arange(most, device="cuda")
    new = starts[1:] - starts[:-1]
    row = (starts[:-1, None] + i).clamp(max=s.tokens - 1)
    q = s.query.view(s.tokens, kv, group, dim)[row].permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * most, dim)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).view(seqs, kv, group, most, -1) * (1.0 / math.sqrt(dim))
    position = (contexts - new)[:, None] + i
    seen = j[None, None, :] <= position[:, :, None]
    if c["window"]:
        seen &= (j[None, None, :] > position[:, :, None] - c["window"]) | (j < c["first"])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    if s.sinks is not None:
        top = torch.maximum(top, s.sinks.view(1, kv, group, 1, 1))
    weights = torch.exp(scores.sub_(top))
    total = weights.sum(-1, keepdim=True)
    if s.sinks is not None:
        total = total + torch.exp(s.sinks.view(1, kv, group, 1, 1) - top)
    out = torch.matmul(weights.view(seqs, kv, group * most, -1), v.contiguous()).view(seqs, kv, group, most, dim) / total
    seq, place = _places(s)
    return out.permute(0, 3, 1, 2, 4)[seq, place - (contexts - new)[seq]].reshape(s.tokens, heads * dim)


def _plain_copy(to, of, moves):
    """pages moves[i][0] of `of` into pages moves[i][1] of `to`; what is not used of the list is behind the rest (-1)"""
    src, dst = moves[:, 0].long(), moves[:, 1].long()
    used = src >= 0
    src, dst = (torch.where(used, x, x[:1].clamp(min=0)) for x in (src, dst))      # (the first once more, or page 0 as it is)
    for t, f in zip(to, of):
        new = f[src]
        t[dst] = torch.where(used[0], new, t[dst]) if t is f else new.to(t.dtype)


def _entered(table, held, references, by, lines):
    """references with `by` added for every page that the given lines of a table hold"""
    j = torch.arange(table.shape[1], device="cuda")
    there = (j[None, :] < held[:, None]) & (table >= 0) & lines[:, None]
    return references.index_add(0, table.clamp(min=0).flatten().long(), (by * there).flatten().to(references.dtype))


def _free(references):
    """the free pages from the lowest on (then the others), and how many there are"""
    free = references == 0
    return torch.sort(free, descending=True, stable=True)[1], free.sum()


def _listed_moves(moves, number, picked, of, to):
    """moves[number] = (of, to) where picked, -1 elsewhere"""
    n = len(moves)
    out = torch.full((n + 1, 2), -1, dtype=torch.int32, device="cuda")
    out[torch.where(picked, number.clamp(max=n), n)] = torch.stack([of, to], dim=1).to(torch.int32)
    moves.copy_(out[:n])


def _plain_fork(s):
    page, table, lens = s.case["page"], s.table, s.lens.long()
    seqs, room = table.shape
    me, j = torch.arange(seqs, device="cuda"), torch.arange(room, device="cuda")
    children = s.children.long()
    last = torch.full((seqs,), -1, device="cuda").scatter_reduce(0, children, torch.arange(len(children), device="cuda"), "amax")
    of = torch.where(last >= 0, s.parents.long()[last.clamp(min=0)], me)
    lowest = torch.full((seqs,), seqs, device="cuda").scatter_reduce(0, of, me, "amin")
    keeper = torch.where(of == me, me, lowest)
    held = (lens + page - 1) // page
    copied = (lens % page != 0)[of] & (keeper[of] != me)
    number = torch.cumsum(copied, 0) - copied.long()
    free, there = _free(s.references)
    fits = copied.sum() <= there
    s.missing.copy_((copied.sum() - there).clamp(min=0)[None])
    fresh = free[number.clamp(max=len(free) - 1)]
    rows = torch.where(j[None, :] < held[of][:, None], table[of], -1)
    begun = rows.gather(1, (held[of] - 1).clamp(min=0)[:, None])[:, 0]
    _listed_moves(s.moves, number, copied & fits, begun, fresh)
    rows = torch.where(copied[:, None] & (j[None, :] == held[of][:, None] - 1), fresh[:, None].to(torch.int32), rows)
    changed = (of != me) & fits
    references = _entered(table, held, s.references, -1, changed)
    references = _entered(rows, held[of], references, 1, changed)
    table.copy_(torch.where(changed[:, None], rows, table))
    s.references.copy_(references)
    s.lens.copy_(torch.where(changed, lens[of], lens))


def _plain_resize(s, lengths):
    page, table, lens = s.case["page"], s.table, s.lens.long()
    seqs, room = table.shape
    j = torch.arange(room, device="cuda")[None, :]
    goal_tokens = torch.where(lengths < 0, lens, lengths.long().clamp(max=room * page))
    held, goal = (lens + page - 1) // page, (goal_tokens + page - 1) // page
    # what is behind the shorter ones' ends is given back
    dropped = (j >= goal[:, None]) & (j < held[:, None])
    references = s.references.index_add(0, table.clamp(min=0).flatten().long(), -(dropped & (table >= 0)).flatten().to(torch.int32))
    entries = torch.where(dropped, -1, table)
    # the longer ones get pages, and one of their own for a shared one that they go on in
    grows = goal_tokens > lens
    end = (held - 1).clamp(min=0)[:, None]
    begun = entries.gather(1, end)[:, 0].long()
    copied = grows & (lens % page != 0) & (begun >= 0) & (references[begun.clamp(min=0)] > 1)
    need = torch.where(grows, goal - held, 0) + copied
    before = torch.cumsum(need, 0) - need
    free, there = _free(references)
    fits = need.sum() <= there
    s.missing.copy_((need.sum() - there).clamp(min=0)[None])
    fresh = free[(before[:, None] + copied[:, None] + j - held[:, None]).clamp(0, len(free) - 1)].to(torch.int32)
    own_page = free[before.clamp(max=len(free) - 1)]
    number = torch.cumsum(copied, 0) - copied.long()
    _listed_moves(s.begun, number, copied & fits, begun, own_page)
    new = grows[:, None] & (j >= held[:, None]) & (j < goal[:, None])
    grown = torch.where(new, fresh, torch.where(copied[:, None] & (j == end), own_page[:, None].to(torch.int32), entries))
    given = torch.where(new | (copied[:, None] & (j == end)), grown, -1)
    more = references.index_add(0, given.clamp(min=0).flatten().long(), (given >= 0).flatten().to(torch.int32))
    more = more.index_add(0, begun.clamp(min=0), -copied.to(torch.int32))
    table.copy_(torch.where(fits, grown, entries))
    s.references.copy_(torch.where(fits, more, references))
    s.lens.copy_(torch.where(grows & ~fits, lens, goal_tokens))


def _plain_compact(s):
    page, room, pages = s.case["page"], len(s.moves), s.pages
    used, number = s.references > 0, torch.arange(pages, device="cuda")
    count = used.sum()
    above, hole = used & (number >= count), ~used & (number < count)
    of = torch.sort(torch.where(above, -number, pages))[1][:room]
    to = torch.sort(torch.where(hole, number, pages))[1][:room]
    picked = torch.arange(len(of), device="cuda") < above.sum()
    _listed_moves(s.moves, torch.arange(len(of), device="cuda"), picked, of, to)
    place = torch.cat([number, number[:1]])                          # (one more for what is not picked)
    place[torch.where(picked, of, pages)] = to
    place = place[:pages]
    held = (s.lens.long() + page - 1) // page
    there = (torch.arange(s.table.shape[1], device="cuda")[None, :] < held[:, None]) & (s.table >= 0)
    s.table.copy_(torch.where(there, place[s.table.clamp(min=0).long()].to(torch.int32), s.table))
    references = torch.cat([s.references, s.references[:1]])
    moved = references[of]
    references[torch.where(picked, of, pages)] = 0
    references[torch.where(picked, to, pages)] = moved
    s.references.copy_(references[:pages])


def _plain_cold(s):
    of, to = s.moves[:, 0].long(), s.moves[:, 1].long()
    for warm, cold, back in zip(s.warm, s.cold, s.back):
        codes, scales = _coded(warm[of].float())
        cold[0][to], cold[1][to] = codes, scales
        at = s.returns[:, 0].long()
        back[s.returns[:, 1].long()] = _values(cold[0][at], cold[1][at]).to(back.dtype)


# ---- the calls -------------------------------------------------------------------------------------------------------------------


def _handles(s):
    """what a program makes once and keeps: the descriptions of the rotation, of the caches with their page table, and of the pool"""
    if s.handles is None:
        from tensorsharp_amd import PagedKVCache, PagePool, RotaryPositions
        c = s.case

        def cache(k, v, table):
            return PagedKVCache(k[0], v[0], table, k[1], v[1]) if isinstance(k, tuple) else PagedKVCache(k, v, table)
        if s.kind == "store":
            s.handles = (cache(s.k, s.v, s.page_table), cache(s.out_k, s.out_v, s.page_table),
                         RotaryPositions(c["rotated"], mode=c["mode"], base=c["base"], freq_factors=s.freq_factors, **s.scaling))
        elif s.kind == "attend":
            s.handles = (cache(s.k, s.v, s.page_table),)
        elif s.kind == "cold":
            s.handles = tuple(cache(*t, s.page_table) for t in (s.warm, s.cold, s.back))
        else:
            pool = PagePool(s.table, s.references, s.lens, c["page"])
            s.handles = (pool, None if s.kind == "turnover" else cache(s.k, s.v, s.table))
    return s.handles


def run(s):
    if own:
        from tensorsharp_amd import HipBasicOps
        handles = _handles(s)
    kind, c = s.kind, s.case
    if kind == "store":
        if not own:
            return _plain_store(s)
        HipBasicOps.RoPEStorePaged(s.query, s.qkv, handles[0], s.row_starts, s.context_lens, handles[2], s.q_norm, s.k_norm, 1e-6)
        HipBasicOps.CopyPages(handles[1], handles[0], s.written)
        return {"query": s.query, "k": s.out_k, "v": s.out_v}
    if kind == "attend":
        if not own:
            return _plain_attend(s)
        HipBasicOps.PagedAttention(s.result, s.query, handles[0], s.row_starts, s.context_lens, 1.0 / math.sqrt(c["dim"]), window=c["window"],
                                   sinks=s.sinks, first=c["first"])
        return s.result
    if kind == "cold":
        if own:
            HipBasicOps.CopyPages(handles[1], handles[0], s.moves)
            HipBasicOps.CopyPages(handles[2], handles[1], s.returns)
        else:
            _plain_cold(s)
        return {"k": s.back[0], "v": s.back[1]}
    out = {"table": s.table, "references": s.references, "lens": s.lens, "missing": s.missing}
    if kind == "fork":
        if own:
            HipBasicOps.ForkSequences(handles[0], s.children, s.parents, s.moves, s.missing)
            HipBasicOps.CopyPages(handles[1], handles[1], s.moves)
        else:
            _plain_fork(s)
            _plain_copy((s.k, s.v), (s.k, s.v), s.moves)
        return {**out, "k": s.k, "v": s.v, "moves": s.moves}
    ended, admitted = s.ended[s.turn % 4], s.admitted[s.turn % 4]
    s.turn += 1
    if own:
        HipBasicOps.ResizeSequences(handles[0], ended, s.begun, s.missing)
        if kind == "compact":
            HipBasicOps.CompactPages(handles[0], s.moves)
            HipBasicOps.CopyPages(handles[1], handles[1], s.moves)
        HipBasicOps.ResizeSequences(handles[0], admitted, s.begun, s.missing)
    else:
        _plain_resize(s, ended)
        if kind == "compact":
            _plain_compact(s)
            _plain_copy((s.k, s.v), (s.k, s.v), s.moves)
        _plain_resize(s, admitted)
    return {**out, "k": s.k, "v": s.v, "moves": s.moves} if kind == "compact" else out


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------------


def work(case):
    kind, page = case["kind"], case["page"]
    if kind == "turnover":
        tokens, _ = _tokens(case)
        ended = [-(-t // page) for t in tokens[::4]]
        return {"bytes": 4 * (4 * sum(ended) + 2 * len(tokens)), "flops": 0}             # their entries and references, taken back and given
    values = case["kv_heads"] * case["dim"]
    if kind == "cold":
        return {"bytes": int(2 * case["moved"] * page * values * 2 * (SIZE[case["type"]] + SIZE["mx4"])), "flops": 0}
    if kind in ("fork", "compact"):
        tokens, _ = _tokens(case)
        counts = [-(-t // page) for t in tokens]
        if kind == "compact":
            moved, lists = sum(counts[::4]) // 2, 4 * sum(counts[::4])
        else:
            each = case["each"]
            moved = sum(each - 1 for t in tokens[::each] if t % page)
            lists = 4 * sum(counts) // each * (each if case["beams"] else each - 1)
        return {"bytes": int(4 * moved * page * values * SIZE[case["type"]] + 4 * lists), "flops": 0}
    news, contexts = _lengths(case)
    tokens, heads, kv, dim = sum(news), case["heads"], case["kv_heads"], case["dim"]
    if kind == "store":
        written = sum(-(-c // page) - (c - n) // page for n, c in zip(news, contexts)) * page * kv * dim
        return {"bytes": int(4 * tokens * (2 * heads + 2 * kv) * dim + 2 * SIZE["mx4"] * (tokens * kv * dim + written) + 4 * written),
                "flops": 3 * tokens * (heads + kv) * case["rotated"]}
    pairs = keys = 0
    window, first = case["window"] or 1 << 40, case["first"]
    for n, ctx in zip(news, contexts):
        p = np.arange(ctx - n, ctx, dtype=np.int64)
        seen = np.minimum(p + 1, window)
        pairs += int((seen + np.minimum(np.maximum(p + 1 - window, 0), first)).sum())
        low = max(0, ctx - n + 1 - window)
        keys += ctx - low + min(first, low)
    return {"bytes": int(8 * tokens * heads * dim + 2 * SIZE[case["type"]] * keys * kv * dim), "flops": 4 * pairs * heads * dim}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------


def _exact_four_bits(x):
    """float64 [.., dim] -> the values that four bits hold of it"""
    grid = torch.tensor(MAGNITUDE, dtype=torch.float64, device=x.device)
    middle = (grid[1:] + grid[:-1]) / 2
    b = x.unflatten(-1, (-1, 32))
    size = b.abs().amax(-1, keepdim=True)
    power = torch.ceil(torch.log2(torch.where(size > 0, size, 1.0) / 7.0))
    power = torch.where(size > 7.0 * 2.0 ** power, power + 1, torch.where(size <= 7.0 * 2.0 ** (power - 1), power - 1, power)).clamp(min=-126.0)
    y = b.abs() / 2.0 ** power
    up, down = torch.bucketize(y, middle, right=True), torch.bucketize(y, middle)
    value = grid[torch.where(up % 2 == 0, up, down)]                 # (they differ in the middle of two codes)
    return torch.where(size < 2.0 ** 127, torch.copysign(value, b) * 2.0 ** power, math.nan).flatten(-2)


def _held(t):
    """float64 values of a cache's tensor, or of its codes and scales"""
    if not isinstance(t, tuple):
        return t.double()
    codes, scales = t
    n = torch.stack([codes % 16, codes // 16], dim=-1).flatten(-2).long()
    e, m = n % 8 // 2, n % 2
    size = torch.where(e == 0, m / 2.0, 2.0 ** (e - 1) * (1 + m / 2.0)).double()
    return (torch.where(n >= 8, -size, size).unflatten(-1, (-1, 32)) * 2.0 ** (scales.double()[..., None] - 127)).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "cold":
        of = s.moves[:, 0].long()
        return {name: _exact_four_bits(t[of].double()) for name, t in zip("kv", s.warm)}
    if s.kind == "attend":
        return _exact_attend(s)
    if s.kind == "store":
        return _exact_store(s)
    return _exact_pages(s)


def _exact_store(s):
    c = s.case
    news, contexts = _lengths(c)
    heads, kv, dim, page, n = c["heads"], c["kv_heads"], c["dim"], c["page"], c["rotated"]
    i = np.arange(n // 2, dtype=np.float64)
    w = c["base"] ** (-2.0 * i / n)
    if s.freq_factors is not None:
        w = w / s.freq_factors.cpu().numpy().astype(np.float64)
    y, size = s.scaling, 1.0
    if y.get("ext_factor"):
        edge = lambda beta: n * np.log(y["original_context"] / (2.0 * np.pi * beta)) / (2.0 * np.log(c["base"]))  # noqa: E731
        low, high = max(np.floor(edge(y["beta_fast"])), 0.0), min(np.ceil(edge(y["beta_slow"])), n - 1.0)
        share = (1.0 - np.minimum(1.0, np.maximum(0.0, (i - low) / max(high - low, 1e-3)))) * y["ext_factor"]
        w = w * y["freq_scale"] * (1.0 - share) + w * share
        size = y["attn_factor"] * (1.0 - 0.1 * np.log(y["freq_scale"]))
    elif y:
        w = w * y["freq_scale"]
    position = torch.cat([torch.arange(t - m, t, device="cuda") for m, t in zip(news, contexts)])
    seq = torch.cat([torch.full((m,), b, device="cuda") for b, m in enumerate(news)])
    turn = size * torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), position.double()[:, None] * torch.from_numpy(w).cuda()[None])[:, None, :]
    x = s.qkv.double().view(s.tokens, -1, dim)
    parts = []
    for at, weight in ((slice(0, heads), s.q_norm), (slice(heads, heads + kv), s.k_norm)):
        part = x[:, at].clone()
        if weight is not None:
            part = part / torch.sqrt((part * part).sum(-1, keepdim=True) / dim + 1e-6) * weight.double()
        pair = (slice(0, n // 2), slice(n // 2, n)) if c["mode"] == 2 else (slice(0, n, 2), slice(1, n, 2))
        z = torch.complex(part[..., pair[0]].contiguous(), part[..., pair[1]].contiguous()) * turn
        part[..., pair[0]], part[..., pair[1]] = z.real, z.imag
        parts.append(part)
    where = (s.page_table.long()[seq, torch.div(position, page, rounding_mode="floor")], torch.remainder(position, page))
    out = {"query": parts[0].reshape(s.tokens, heads * dim)}
    for name, cache, new in (("k", s.k, parts[1]), ("v", s.v, x[:, heads + kv:])):
        whole = _held(cache)
        whole[where] = _exact_four_bits(new)
        out[name] = whole[s.written[:, 0].long()]
    return out


def _exact_attend(s):
    c = s.case
    news, contexts = _lengths(c)
    heads, kv, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    table = s.page_table.long()
    out = torch.zeros((s.tokens, heads, dim), dtype=torch.float64, device="cuda")
    row = 0
    for b, (n, ctx) in enumerate(zip(news, contexts)):
        j = torch.arange(ctx, device="cuda")
        at = (table[b, torch.div(j, page, rounding_mode="floor")], torch.remainder(j, page))
        k, v = (_held((t[0][at], t[1][at]) if isinstance(t, tuple) else t[at]) for t in (s.k, s.v))
        back = torch.arange(ctx - n, ctx, device="cuda")[:, None] - j[None, :]      # how far behind the token a key lies
        hidden = back < 0
        if c["window"]:
            hidden = hidden | ((back >= c["window"]) & (j[None, :] >= c["first"]))
        for h in range(heads):
            g = h // (heads // kv)
            q = s.query[row:row + n].view(n, heads, dim)[:, h].double()
            z = (q @ k[:, g].t().contiguous()) / math.sqrt(dim)
            z[hidden] = -math.inf
            if s.sinks is not None:
                z = torch.cat([z, s.sinks[h].double().expand(n, 1)], dim=1)
            z = torch.exp(z - z.max(1, keepdim=True).values)
            out[row:row + n, h] = (z[:, :ctx] @ v[:, g].contiguous()) / z.sum(1, keepdim=True)
        row += n
    return out.view(s.tokens, heads * dim)


def _exact_pages(s):
    """the lists as a program with a heap of pages would keep them, page by page"""
    page, kind = s.case["page"], s.kind
    lens, references = s.lens.tolist(), s.references.tolist()
    table = s.table.cpu().numpy()
    rows = [list(map(int, r[:-(-n // page)])) for r, n in zip(table, lens)]
    moves = []

    def free_pages():
        return [p for p, r in enumerate(references) if r == 0]

    def resize(goals):
        for i, n in enumerate(goals):
            if 0 <= n < lens[i]:
                for p in rows[i][-(-n // page):]:
                    references[p] -= 1
                rows[i], lens[i] = rows[i][:-(-n // page)], n
        free = iter(free_pages())
        for i, n in enumerate(goals):
            if n > lens[i]:                                          # (the cases' sequences share no pages, and there are enough)
                new = [next(free) for _ in range(-(-n // page) - len(rows[i]))]
                for p in new:
                    references[p] += 1
                rows[i], lens[i] = rows[i] + new, n
    if kind == "fork":
        parent = list(range(len(rows)))
        for c, p in zip(s.children.tolist(), s.parents.tolist()):
            parent[c] = p
        taken, free, old_rows, old_lens = {p for i, p in enumerate(parent) if i == p}, iter(free_pages()), [list(r) for r in rows], list(lens)
        fresh = []
        for i, p in enumerate(parent):
            lens[i] = old_lens[p]
            if i == p:
                continue
            rows[i] = list(old_rows[p])
            if old_lens[p] % page:
                if p in taken:
                    fresh.append(next(free))
                    moves.append((rows[i][-1], fresh[-1]))
                    rows[i][-1] = fresh[-1]
                taken.add(p)
        count = np.bincount([p for r in rows for p in r], minlength=len(references))
        references = [int(c) for c in count]
    else:
        resize(s.ended[0].tolist())
        if kind == "compact":
            used = sum(r > 0 for r in references)
            holes = [p for p in range(used) if references[p] == 0]
            tops = [p for p in range(len(references) - 1, used - 1, -1) if references[p] > 0]
            moves = list(zip(tops, holes))
            for of, to in moves:
                references[to], references[of] = references[of], 0
            new = dict(moves)
            rows = [[new.get(p, p) for p in r] for r in rows]
        resize(s.admitted[0].tolist())
    out = np.full(table.shape, -1, dtype=np.int32)
    for i, r in enumerate(rows):
        out[i, :len(r)] = r
    answer = {"table": out, "references": np.array(references, dtype=np.int32), "lens": np.array(lens, dtype=np.int32), "missing": np.zeros(1, dtype=np.int32)}
    if kind == "turnover":
        return answer
    filled = np.full(s.moves.shape, -1, dtype=np.int32)
    filled[:len(moves)] = np.array(moves, dtype=np.int32).reshape(-1, 2)
    k, v = s.k.double(), s.v.double()
    if moves:
        of, to = (torch.tensor(x, device="cuda") for x in zip(*moves))
        k[to], v[to] = k[of], v[of]
    return {**answer, "k": k, "v": v, "moves": filled}
