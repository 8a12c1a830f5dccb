"""GPU: attention of new tokens over a paged cache against its definition in 64 bits.

Bounds.  A score sums dim products in 32 bits, its worst case (dim + 8) 2^-24 of scale sum |q k|; the parts that q is cut into leave 2^-21 of
that, the exponent's argument and the exponential 4 x 2^-24 (1 + |s|).  An error e in the scores moves a result by at most 2 e sum p |v|, and the
weighted sum rounds 2^-20 of sum p |v| (parts of the weights 2^-20.. 2^-21, sums over tiles).  Held element by element.  That is the
worst case; roundings of random sign leave 2^-24 sqrt(dim) times the size of a score (2 where queries are N(0, 2) and keys N(0, 1)) and less than
that for the rest.  Relative to the norm of the result three times that is held as well (4e-6 at a size of 2 and 128 dimensions), which one
16-bit rounding of q or of the weights (1e-4) would break."""
import numpy as np
import pytest

import paged_oracle as po

pytestmark = pytest.mark.gpu


def starts_of(news, torch):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(news)]).astype(np.int32)).cuda()


def run(hip, torch, c, q, news, contexts, scale, window=0, sinks=None, rows=None, table=None):
    from tensorsharp_amd import PagedKVCache
    rows = sum(news) if rows is None else rows
    out = torch.full((rows, q.shape[1]), 7.5, device="cuda")
    lens = torch.tensor(contexts, dtype=torch.int32, device="cuda")
    hip.PagedAttention(out, q, PagedKVCache(c.k, c.v, c.table_dev if table is None else table), starts_of(news, torch), lens, scale, window=window,
                       sinks=sinks)
    return out


def check(out, c, q, news, contexts, heads, dim, scale, window, sinks, present=None, size_of_scores=2.0):
    got, at = out.cpu().numpy().astype(np.float64).reshape(len(out), heads, dim), 0
    qs = q.cpu().numpy().astype(np.float64).reshape(len(q), heads, dim)
    errors, refs = [], []
    for s, (n, ctx) in enumerate(zip(news, contexts)):
        if n == 0:
            continue
        k, v = c.rows(s, contexts)
        group = heads // k.shape[1]
        ref, size = po.attend(qs[at:at + n], np.nan_to_num(k), np.nan_to_num(v), np.arange(ctx - n, ctx), scale, window,
                              None if sinks is None else sinks.cpu().numpy(), None if present is None else present[s])
        most = np.zeros((n, heads))
        for h in range(heads):                                       # the largest scale sum |q k| of a row
            most[:, h] = abs(scale) * (np.abs(qs[at:at + n, h]) @ np.abs(np.nan_to_num(k[:, h // group])).T).max(1, initial=0.0)
        e = most * ((dim + 8) * 2.0 ** -24 + 2.0 ** -21 + 4 * 2.0 ** -24) + 4 * 2.0 ** -24
        d = np.abs(got[at:at + n] - ref)
        assert np.all(d <= (2 * e[..., None] + 2.0 ** -20) * size), (s, float((d / np.maximum(size, 1e-30)).max()))
        errors.append(d.ravel())
        refs.append(ref.ravel())
        at += n
    if refs:
        r = np.linalg.norm(np.concatenate(refs))
        assert np.linalg.norm(np.concatenate(errors)) <= 3 * 2.0 ** -24 * np.sqrt(max(dim, 128)) * size_of_scores * max(r, 1e-30)


CASES = [
    # heads, kv heads, dim, type, page, order, contexts, new tokens, window, sinks
    (32, 8, 128, "float16", 16, "token", [1], [1], 0, False),
    (32, 8, 128, "float16", 16, "token", [777, 1, 64, 33, 1500], [1, 1, 1, 1, 1], 0, False),
    (32, 8, 128, "float16", 64, "head", [300], [300], 0, False),
    (8, 8, 128, "float16", 1, "token", [130, 70], [70, 2], 0, True),
    (8, 1, 128, "bfloat16", 24, "token", [200, 513, 40], [150, 1, 40], 128, True),
    (64, 8, 64, "bfloat16", 16, "head", [700, 260, 5], [65, 1, 5], 100, True),
    (6, 2, 64, "float16", 5, "token", [97, 31, 2], [33, 31, 1], 0, False),
    (7, 1, 80, "float16", 100, "head", [250, 90], [9, 33], 0, True),
    (5, 1, 96, "bfloat16", 32, "token", [129, 300], [128, 3], 17, False),
    (4, 4, 112, "float32", 7, "token", [90, 40], [21, 40], 0, False),
    (16, 2, 128, "float32", 4096, "head", [333], [100], 0, False),
    (3, 3, 192, "float16", 16, "token", [70, 300], [70, 1], 1, True),
    (8, 2, 256, "float16", 16, "head", [150, 260], [65, 1], 0, False),
    (8, 2, 256, "bfloat16", 33, "token", [150, 260], [40, 1], 0, False),
    (4, 2, 256, "float32", 16, "token", [100, 260], [33, 2], 50, True),
    (2, 1, 16, "float16", 3, "token", [50, 10], [17, 10], 0, False),
    (12, 12, 48, "bfloat16", 256, "head", [300, 1], [129, 1], 0, False),
    (36, 4, 160, "float16", 16, "token", [100], [20], 0, False),
    (6, 2, 192, "float32", 16, "head", [140, 90], [50, 1], 0, False),
    (8, 1, 176, "bfloat16", 64, "token", [200, 60], [30, 3], 70, True),
]


@pytest.mark.parametrize("heads,kv,dim,dtype,page,order,contexts,news,window,sunk", CASES)
def test_attention(hip, heads, kv, dim, dtype, page, order, contexts, news, window, sunk):
    import torch
    rng = np.random.default_rng(heads * dim + page)
    c = po.Cache(torch, rng, contexts, page, kv, dim, getattr(torch, dtype), order)
    rows = sum(news)
    q = torch.from_numpy((2.0 * rng.standard_normal((rows + 2, heads * dim))).astype(np.float32)).cuda()
    sinks = torch.from_numpy(rng.standard_normal(heads).astype(np.float32)).cuda() if sunk else None
    scale = 1.0 / np.sqrt(dim)
    out = run(hip, torch, c, q, news, contexts, scale, window, sinks, rows=rows + 2)
    assert torch.all(out[rows:] == 7.5)                              # rows of no sequence
    check(out[:rows], c, q[:rows], news, contexts, heads, dim, scale, window, sinks)
    same = q.clone()                                                 # in place
    from tensorsharp_amd import PagedKVCache
    hip.PagedAttention(same, same, PagedKVCache(c.k, c.v, c.table_dev), starts_of(news, torch), torch.tensor(contexts, dtype=torch.int32, device="cuda"),
                       scale, window=window, sinks=sinks)
    assert torch.equal(same[:rows], out[:rows]) and torch.equal(same[rows:], q[rows:])


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("dim", [192, 256])
@pytest.mark.parametrize("news,contexts", [([1, 7, 1], [300, 129, 31]), ([130, 5], [700, 64]), ([20], [1200])])
def test_large_heads(hip, dtype, dim, news, contexts):
    """the sizes whose rows and accumulators fill the registers, with short and long tiles, cut and whole"""
    import torch
    rng = np.random.default_rng(dim + len(news))
    heads, kv = 6, 2
    c = po.Cache(torch, rng, contexts, 16, kv, dim, getattr(torch, dtype))
    q = torch.from_numpy((2.0 * rng.standard_normal((sum(news), heads * dim))).astype(np.float32)).cuda()
    for window in (0, 150):
        out = run(hip, torch, c, q, news, contexts, dim ** -0.5, window)
        check(out, c, q, news, contexts, heads, dim, dim ** -0.5, window, None)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("news,contexts", [([1, 1], [9000, 4100]), ([40], [5000]), ([2, 0, 70], [3001, 50, 2999])])
def test_long_contexts(hip, dtype, news, contexts):
    """few rows and many keys: the keys are shared out and the parts joined"""
    import torch
    rng = np.random.default_rng(len(contexts))
    heads, kv, dim = 8, 2, 128
    c = po.Cache(torch, rng, contexts, 16, kv, dim, getattr(torch, dtype))
    q = torch.from_numpy((2.0 * rng.standard_normal((sum(news), heads * dim))).astype(np.float32)).cuda()
    sinks = torch.from_numpy(rng.standard_normal(heads).astype(np.float32)).cuda()
    for window, sink in ((0, None), (2100, sinks)):
        out = run(hip, torch, c, q, news, contexts, dim ** -0.5, window, sink)
        check(out, c, q, news, contexts, heads, dim, dim ** -0.5, window, sink)
        assert torch.equal(out, run(hip, torch, c, q, news, contexts, dim ** -0.5, window, sink))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("spread", [0.0, 30.0])
def test_weights_of_very_different_sizes(hip, dtype, spread):
    """scores that grow or fall along the keys by hundreds (the running maximum moves at every step, or never), a single key that takes all,
    queries far outside the range of 16-bit floats"""
    import torch
    rng = np.random.default_rng(5)
    heads, kv, dim, ctx, n = 4, 2, 64, 700, 35
    c = po.Cache(torch, rng, [ctx], 16, kv, dim, getattr(torch, dtype))
    for sign in (1.0, -1.0):
        slope = (sign * spread * np.arange(ctx) / ctx).astype(np.float32)
        k = c.host[0]
        p = np.arange(ctx)
        k[c.table[0, p // 16], p % 16, :, 0] = slope[:, None]
        c.k = torch.from_numpy(k).cuda().to(c.dtype)
        q = rng.standard_normal((n, heads, dim)).astype(np.float32)
        q[..., 0] = 8.0
        qd = torch.from_numpy(q.reshape(n, -1)).cuda()
        for by, scale in ((1.0, 0.5), (1e9, 0.5e-9), (1e-9, 0.5e9)):
            out = run(hip, torch, c, qd * by, [n], [ctx], scale)
            check(out, c, qd * by, [n], [ctx], heads, dim, scale, 0, None, size_of_scores=max(2.0, 0.5 * 8.0 * spread))


def test_pages_that_are_not_there_hold_nothing(hip):
    import torch
    rng = np.random.default_rng(8)
    heads, kv, dim, ctx, n = 8, 2, 128, 400, 37
    c = po.Cache(torch, rng, [ctx, 30], 16, kv, dim, torch.float16)
    bad = c.table.copy()
    bad[0, [0, 3, 7, 24]] = [-1, len(c.k), 2 ** 31 - 1, -2 ** 31]
    bad[1] = -5
    present = [np.ones(ctx, bool), np.zeros(30, bool)]
    for p in (0, 3, 7, 24):
        present[0][16 * p:16 * p + 16] = False
    c.host = None
    q = torch.from_numpy(rng.standard_normal((n + 2, heads * dim)).astype(np.float32)).cuda()
    for sinks in (None, torch.zeros(heads, device="cuda")):
        out = run(hip, torch, c, q, [n, 2], [ctx, 30], 0.1, 0, sinks, table=torch.from_numpy(bad).cuda())
        assert torch.all(out[n:] == 0)                               # nothing to see: zero, not NaN
        check(out, c, q, [n, 2], [ctx, 30], heads, dim, 0.1, 0, sinks, present)


def test_rows_that_see_nothing(hip):
    """more new tokens than the context holds: the first ones are before the sequence; a context beyond the page table: what is not there is not
    seen"""
    import torch
    rng = np.random.default_rng(9)
    heads, kv, dim = 4, 2, 64
    c = po.Cache(torch, rng, [20, 16], 8, kv, dim, torch.float16)
    q = torch.from_numpy(rng.standard_normal((34, heads * dim)).astype(np.float32)).cuda()
    out = run(hip, torch, c, q, [30, 4], [20, 60], 0.2)
    assert torch.all(out[:10] == 0)
    got = out.cpu().numpy().reshape(34, heads, dim)
    k, v = c.rows(0)
    ref, _ = po.attend(q[10:30].cpu().numpy().reshape(20, heads, dim), k, v, np.arange(20), 0.2)
    assert np.abs(got[10:30] - ref).max() < 1e-5
    k, v = c.rows(1)                                                 # positions 56 .. 59 of 16 that are there
    ref, _ = po.attend(q[30:].cpu().numpy().reshape(4, heads, dim), k, v, np.arange(56, 60), 0.2)
    assert np.abs(got[30:] - ref).max() < 1e-5
    assert torch.all(run(hip, torch, c, q, [30, 4], [-7, 0], 0.2) == 0)


def test_strided_tensors_and_a_cache_within_a_larger_one(hip):
    import torch
    from tensorsharp_amd import PagedKVCache
    rng = np.random.default_rng(10)
    heads, kv, dim, ctx, n = 6, 3, 64, 130, 50
    c = po.Cache(torch, rng, [ctx], 16, kv, dim, torch.bfloat16)
    both = torch.full((len(c.k), 2, 16, kv + 1, dim + 8), float("nan"), device="cuda", dtype=torch.bfloat16)   # keys and values of a page side by side
    both[:, 0, :, :kv, :dim], both[:, 1, :, :kv, :dim] = c.k, c.v
    wide = torch.zeros((n, heads * dim + 12), device="cuda")
    q = torch.from_numpy(rng.standard_normal((n, heads * dim)).astype(np.float32)).cuda()
    wide[:, 4:4 + heads * dim] = q
    out = torch.full((n, heads * dim + 20), 7.5, device="cuda")
    table = torch.full((1, 40), -1, dtype=torch.int32, device="cuda")
    table[:, :c.table.shape[1]] = c.table_dev
    hip.PagedAttention(out[:, 8:8 + heads * dim], wide[:, 4:4 + heads * dim], PagedKVCache(both[:, 0, :, :kv, :dim], both[:, 1, :, :kv, :dim], table),
                       starts_of([n], torch), torch.tensor([ctx], dtype=torch.int32, device="cuda"), 0.125)
    check(out[:, 8:8 + heads * dim], c, q, [n], [ctx], heads, dim, 0.125, 0, None)
    assert torch.all(out[:, :8] == 7.5) and torch.all(out[:, 8 + heads * dim:] == 7.5)


def test_many_sequences(hip):
    """more than a wavefront has lanes, some without new tokens"""
    import torch
    rng = np.random.default_rng(12)
    heads, kv, dim = 4, 1, 64
    contexts = [int(v) for v in rng.integers(1, 90, 150)]
    news = [min(c, int(v)) for c, v in zip(contexts, rng.integers(0, 4, 150))]
    c = po.Cache(torch, rng, contexts, 8, kv, dim, torch.float16)
    q = torch.from_numpy(rng.standard_normal((sum(news), heads * dim)).astype(np.float32)).cuda()
    out = run(hip, torch, c, q, news, contexts, 0.125)
    check(out, c, q, news, contexts, heads, dim, 0.125, 0, None)


def test_offsets_beyond_32_bits(hip):
    """a cache of 5 GiB per tensor, the pages at its end"""
    import torch
    from tensorsharp_amd import PagedKVCache
    rng = np.random.default_rng(13)
    heads, kv, dim, ctx = 4, 2, 128, 70
    c = po.Cache(torch, rng, [ctx], 16, kv, dim, torch.float16)
    pages = (5 << 30) // (16 * kv * dim * 2)
    k, v = (torch.empty((pages, 16, kv, dim), dtype=torch.float16, device="cuda") for _ in range(2))
    table = c.table_dev + (pages - len(c.k))
    for big, small in ((k, c.k), (v, c.v)):
        big[pages - len(small):] = small
    q = torch.from_numpy(rng.standard_normal((20, heads * dim)).astype(np.float32)).cuda()
    out = torch.zeros_like(q)
    hip.PagedAttention(out, q, PagedKVCache(k, v, table), starts_of([20], torch), torch.tensor([ctx], dtype=torch.int32, device="cuda"), 0.1)
    check(out, c, q, [20], [ctx], heads, dim, 0.1, 0, None)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("n,window,dim,ctx", [(100, 0, 64, 300), (100, 40, 64, 300), (3, 0, 128, 300), (3, 60, 96, 300), (70, 0, 256, 300), (3, 0, 192, 3001),
                                              (90, 0, 128, 2500), (1, 0, 128, 300), (1, 0, 64, 5000), (1, 7, 80, 300)])
def test_what_is_no_number_reaches_the_rows_that_see_it_only(hip, dtype, n, window, dim, ctx):
    """infinities and NaN among the keys and values of tokens that some rows see and earlier (or, behind a window, later) ones do not; one
    token sees them all (an infinite key gives a weight of zero or no number, by the sign of the query)"""
    import torch
    rng = np.random.default_rng(n)
    heads, kv = 8, 2
    c = po.Cache(torch, rng, [ctx], 16, kv, dim, getattr(torch, dtype))

    def poison(host, token, head, d, value):
        host[c.table[0, token // 16], token % 16, head, d] = value
    poison(c.host[1], ctx - 2, 0, 3, np.inf)
    poison(c.host[1], ctx - 2, 0, dim - 1, -np.inf)
    poison(c.host[1], ctx - n // 2 - 1, 1, 0, np.nan)
    poison(c.host[0], ctx - 1, 1, slice(None) if n > 1 else 2, np.nan if n > 1 else np.inf)
    if window:
        poison(c.host[1], ctx - window - 1, 1, 5, np.inf)
    c.k, c.v = (torch.from_numpy(t).cuda().to(c.dtype) for t in c.host)
    q = torch.from_numpy(rng.standard_normal((n, heads * dim)).astype(np.float32)).cuda()
    out = run(hip, torch, c, q, [n], [ctx], dim ** -0.5, window).cpu().numpy().reshape(n, heads, dim)
    k, v = c.rows(0)
    with np.errstate(invalid="ignore"):
        ref, _ = po.attend(q.cpu().numpy().reshape(n, heads, dim), k, v, np.arange(ctx - n, ctx), dim ** -0.5, window)
    fine = np.isfinite(ref)
    assert 0 < fine.sum() < fine.size
    assert np.array_equal(np.isnan(ref), np.isnan(out)) and np.array_equal(ref[np.isinf(ref)], out[np.isinf(ref)])
    assert np.linalg.norm(out[fine] - ref[fine]) <= 4e-6 * np.linalg.norm(ref[fine])
