"""GPU: attention over a cache in four bits against its definition in 64 bits over the values that the codes stand for.

Bounds.  A row of q goes in as five terms of blocks of 32: a term's rounding leaves at most half a step of 0.5 beside a block's largest of more than
3.75 units, a fifteenth of it, so 15^-5 of the block's largest is lost per value.  Sums of dim products in 32 bits leave (dim + 8) 2^-24 of scale sum |q k| at
worst, the exponent's argument and the exponential 4 x 2^-24 (1 + |s|).  An error e in the scores moves a result by at most 2 e sum p |v|, and the weighted sum
rounds 2^-20 of sum p |v|.  Held element by element; relative to the norm of the result, as test_gpu_paged_attention.py derives it, 3 2^-24 sqrt(max(dim, 128))
times the size of the scores."""
import numpy as np
import pytest

import mx4_oracle as mx
from attention_oracle import FourBits, attend

pytestmark = pytest.mark.gpu


def starts_of(news, torch):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(news)]).astype(np.int32)).cuda()


def run(hip, torch, c, q, news, contexts, scale, window=0, first=0, sinks=None, table=None):
    out = torch.full((len(q), q.shape[1]), 7.5, device="cuda")
    lens = torch.tensor(contexts, dtype=torch.int32, device="cuda")
    hip.PagedAttention(out, q, c.cache(table), starts_of(news, torch), lens, scale, window=window, sinks=sinks, first=first)
    return out


def check(out, c, q, news, contexts, heads, dim, scale, window=0, first=0, sinks=None, present=None, size_of_scores=2.0, terms=True):
    got, at = out.cpu().numpy().astype(np.float64).reshape(len(out), heads, dim), 0
    qs = q.cpu().numpy().astype(np.float64).reshape(len(q), heads, dim)
    errors, refs = [], []
    for s, (n, ctx) in enumerate(zip(news, contexts)):
        if n == 0:
            continue
        k, v = (np.nan_to_num(t) for t in c.rows(s, contexts))
        group = heads // k.shape[1]
        x = qs[at:at + n]
        ref, size = attend(x, k, v, np.arange(ctx - n, ctx), scale, window, first, None if sinks is None else sinks.cpu().numpy(),
                           None if present is None else present[s])
        e = np.zeros((n, heads))
        for h in range(heads):
            keys = np.abs(k[:, h // group])
            most = abs(scale) * (np.abs(x[:, h]) @ keys.T).max(1, initial=0.0)
            e[:, h] = most * ((dim + 8) * 2.0 ** -24 + 4 * 2.0 ** -24) + 4 * 2.0 ** -24
            if terms:
                block = np.abs(x[:, h]).reshape(n, -1, 32).max(-1)
                e[:, h] += abs(scale) * 15.0 ** -5 * (block @ keys.reshape(len(keys), -1, 32).sum(-1).T).max(1, initial=0.0)
            else:
                e[:, h] += most * 2.0 ** -21
        d = np.abs(got[at:at + n] - ref)
        assert np.all(d <= (2 * e[..., None] + 2.0 ** -20) * size), (s, float((d / np.maximum(size, 1e-30)).max()))
        errors.append(d.ravel())
        refs.append(ref.ravel())
        at += n
    if refs:
        r = np.linalg.norm(np.concatenate(refs))
        assert np.linalg.norm(np.concatenate(errors)) <= 3 * 2.0 ** -24 * np.sqrt(max(dim, 128)) * size_of_scores * max(r, 1e-30)


CASES = [
    # heads, kv heads, dim, page, order, contexts, new tokens, window, first positions, sinks
    (32, 8, 128, 16, "token", [1], [1], 0, 0, False),
    (32, 8, 128, 16, "token", [777, 1, 64, 33, 1500], [1, 1, 1, 1, 1], 0, 0, False),
    (32, 8, 128, 64, "head", [300], [300], 0, 0, False),
    (8, 8, 128, 1, "token", [130, 70], [70, 2], 0, 0, True),
    (8, 1, 128, 24, "token", [200, 513, 40], [150, 1, 40], 128, 0, True),
    (64, 8, 64, 16, "head", [700, 260, 5], [65, 1, 5], 100, 7, True),
    (6, 2, 64, 5, "token", [97, 31, 2], [33, 31, 1], 0, 0, False),
    (7, 1, 32, 100, "head", [250, 90], [9, 33], 0, 0, True),
    (5, 1, 96, 32, "token", [129, 300], [128, 3], 17, 4, False),
    (4, 4, 160, 7, "token", [90, 40], [21, 40], 0, 0, False),
    (16, 2, 128, 4096, "head", [333], [100], 0, 0, False),
    (3, 3, 192, 16, "token", [70, 300], [70, 1], 1, 1, True),
    (8, 2, 256, 16, "head", [150, 260], [65, 1], 0, 0, False),
    (8, 2, 256, 33, "token", [150, 260], [40, 1], 60, 65, False),
    (24, 1, 128, 16, "token", [400, 90], [1, 1], 0, 0, False),
    (8, 2, 224, 3, "token", [50, 10], [17, 10], 0, 0, False),
    (20, 2, 96, 16, "head", [500], [2], 300, 3, False),
    (2, 2, 64, 256, "head", [300, 1], [129, 1], 0, 0, False),
    (16, 1, 64, 16, "token", [200, 60], [2, 1], 70, 2, True),
    (2, 1, 32, 1, "token", [70, 7], [1, 7], 3, 200, False),
]


@pytest.mark.parametrize("heads,kv,dim,page,order,contexts,news,window,first,sunk", CASES)
def test_attention(hip, heads, kv, dim, page, order, contexts, news, window, first, sunk):
    import torch
    rng = np.random.default_rng(heads * dim + page)
    c = FourBits(torch, rng, contexts, page, kv, dim, order)
    rows = sum(news)
    q = torch.from_numpy((2.0 * rng.standard_normal((rows + 2, heads * dim))).astype(np.float32)).cuda()
    sinks = torch.from_numpy(rng.standard_normal(heads).astype(np.float32)).cuda() if sunk else None
    scale = 1.0 / np.sqrt(dim)
    out = run(hip, torch, c, q, news, contexts, scale, window, first, sinks)
    assert torch.all(out[rows:] == 7.5)                              # rows of no sequence
    check(out[:rows], c, q[:rows], news, contexts, heads, dim, scale, window, first, sinks)
    same = q.clone()                                                 # in place
    hip.PagedAttention(same, same, c.cache(), starts_of(news, torch), torch.tensor(contexts, dtype=torch.int32, device="cuda"), scale, window=window,
                       sinks=sinks, first=first)
    assert torch.equal(same[:rows], out[:rows]) and torch.equal(same[rows:], q[rows:])


@pytest.mark.parametrize("dim,heads,kv", [(128, 8, 2), (256, 4, 1), (64, 16, 4), (192, 6, 2), (96, 5, 1)])
@pytest.mark.parametrize("news,contexts", [([1], [7000]), ([1, 2, 1], [2500, 90, 4001]), ([9], [3001]), ([40], [2600]), ([300, 1], [2800, 1900])])
def test_keys_cut_into_pieces(hip, dim, heads, kv, news, contexts):
    import torch
    rng = np.random.default_rng(dim + len(news))
    c = FourBits(torch, rng, contexts, 16, kv, dim, "head")
    q = torch.from_numpy((2.0 * rng.standard_normal((sum(news), heads * dim))).astype(np.float32)).cuda()
    for window, first in ((0, 0), (1500, 0), (1500, 130)):
        out = run(hip, torch, c, q, news, contexts, 1.0 / np.sqrt(dim), window, first)
        check(out, c, q, news, contexts, heads, dim, 1.0 / np.sqrt(dim), window, first)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0, 1e-30])
def test_scales(hip, scale):
    import torch
    rng = np.random.default_rng(5)
    c = FourBits(torch, rng, [70, 200], 16, 2, 64)
    q = torch.from_numpy(rng.standard_normal((41, 4 * 64)).astype(np.float32)).cuda()
    out = run(hip, torch, c, q, [1, 40], [70, 200], scale)
    check(out, c, q, [1, 40], [70, 200], 4, 64, scale, size_of_scores=max(2.0, 8 * abs(scale)))


def test_what_no_row_sees_and_pages_that_are_not_there(hip):
    """sequences without rows, without tokens, entries that are no pages: neither read nor counted; a row that sees nothing is zero"""
    import torch
    rng = np.random.default_rng(6)
    contexts, news = [100, 50, 300, 40, 130], [3, 0, 1, 1, 60]
    c = FourBits(torch, rng, contexts, 16, 2, 128)
    table = c.table.copy()
    table[0, 2], table[2, 0], table[2, 18], table[4, 1] = -1, 2 ** 31 - 1, -2 ** 31, 10 ** 6
    table[3, :] = -1
    present = []
    for s, n in enumerate(contexts):
        p = np.arange(n)
        present.append((table[s, p // 16] >= 0) & (table[s, p // 16] < c.codes[0].shape[0]))
    q = torch.from_numpy(rng.standard_normal((65, 8 * 128)).astype(np.float32)).cuda()
    for window, first in ((0, 0), (20, 0), (20, 5)):
        out = run(hip, torch, c, q, news, contexts, 0.1, window, first, table=torch.from_numpy(table).cuda())
        check(out, c, q, news, contexts, 8, 128, 0.1, window, first, present=present)
        assert torch.all(out[4] == 0)
    empty = run(hip, torch, c, q[:2], [1, 1, 0, 0, 0], [0, -3, 0, 0, 0], 0.1)
    assert torch.all(empty == 0)


@pytest.mark.parametrize("kind", ["values", "keys"])
@pytest.mark.parametrize("news", [[1, 1], [20, 60]])
def test_blocks_of_nan_reach_only_rows_that_see_them(hip, kind, news):
    import torch
    rng = np.random.default_rng(8)
    contexts, dim, heads, kv = [300, 400], 128, 4, 2
    bad = {0: [100, 285], 1: [10, 380, 395]}

    def make(i, s, n):
        x = rng.standard_normal((n, kv, dim))
        if i == (kind == "values"):
            x[bad[s], 1, 40] = np.nan
        return x
    c = FourBits(torch, rng, contexts, 16, kv, dim, make=make)
    q = torch.from_numpy(rng.standard_normal((sum(news), heads * dim)).astype(np.float32)).cuda()
    for window, first in ((0, 0), (50, 0), (50, 12), (5, 0)):
        out = run(hip, torch, c, q, news, contexts, 0.1, window, first).cpu().numpy().reshape(-1, heads, dim)
        clean = FourBits.__new__(FourBits)
        clean.__dict__.update(c.__dict__)
        row = 0
        for s, n in enumerate(news):
            k, v = (np.nan_to_num(t) for t in c.rows(s))
            p = np.arange(contexts[s] - n, contexts[s])
            sees = np.array([any((b <= x) and (not window or b > x - window or b < first) for b in bad[s]) for x in p])
            ref, size = attend(q.cpu().numpy()[row:row + n].reshape(n, heads, dim), k, v, p, 0.1, window, first)
            got = out[row:row + n]
            assert np.all(np.abs(got[:, :2] - ref[:, :2]) <= 1e-5 * size[:, :2] + 1e-7)
            assert np.all(np.abs(got[~sees][:, 2:] - ref[~sees][:, 2:]) <= 1e-5 * size[~sees][:, 2:] + 1e-7)
            if kind == "keys":
                assert np.all(np.isnan(got[sees][:, 2:]))
            else:
                assert np.all(np.isnan(got[sees][:, 2:, 32:64])) and np.all(np.isfinite(got[sees][:, 2:, :32])) and np.all(np.isfinite(got[sees][:, 2:, 64:]))
                rest = np.r_[0:32, 64:128]
                assert np.all(np.abs(got[sees][:, 2:][..., rest] - ref[sees][:, 2:][..., rest]) <= 1e-5 * size[sees][:, 2:][..., rest] + 1e-7)
            row += n


@pytest.mark.parametrize("news", [[1], [50]])
def test_sizes_of_values_and_scores(hip, news):
    """values next to the largest and smallest that a block may hold, a first key that takes nearly all and holds nothing, scores far apart"""
    import torch
    rng = np.random.default_rng(9)
    n, dim, heads, kv = 700, 64, 4, 2
    q = torch.from_numpy(rng.standard_normal((news[0], heads * dim)).astype(np.float32)).cuda()
    for size in (2.0 ** 124, 2.0 ** -110):
        c = FourBits(torch, rng, [n], 16, kv, dim, make=lambda i, s, m: rng.standard_normal((m, kv, dim)) * (1.0 if i == 0 else size / 8))
        out = run(hip, torch, c, q, news, [n], 0.1)
        assert torch.isfinite(out).all()
        check(out, c, q, news, [n], heads, dim, 0.1)
    ahead = np.zeros((n, kv, dim))

    def make(i, s, m):
        x = rng.standard_normal((m, kv, dim)) * (0.01 if i == 0 else 1.0)
        x[0] = 4.0 if i == 0 else 0.0
        return x
    c = FourBits(torch, rng, [n], 16, kv, dim, make=make)
    one = torch.full((news[0], heads * dim), 1.0, device="cuda")
    for folds in (8.0, 20.0, 30.0):                                  # that the first key lies above the others
        scale = folds / (4.0 * dim)
        out = run(hip, torch, c, one, news, [n], scale)
        check(out, c, one, news, [n], heads, dim, scale, size_of_scores=folds)
    assert ahead.shape == (n, kv, dim)


def test_every_code_and_power_as_key_and_value(hip):
    """one key at a time with all codes: the result is the value, whatever its power; scores of all codes against one query"""
    import torch
    codes = np.arange(256, dtype=np.uint8)
    powers = np.array([1, 2, 60, 100, 127, 140, 200, 250, 252], dtype=np.uint8)
    n, dim = len(powers) * 16, 32
    from tensorsharp_amd import PagedKVCache
    v = np.zeros((n, 1, 1, 16), dtype=np.uint8)
    vs = np.zeros((n, 1, 1, 1), dtype=np.uint8)
    for i, p in enumerate(powers):
        for j in range(16):
            v[16 * i + j, 0, 0] = codes[16 * j:16 * j + 16]
            vs[16 * i + j] = p
    k, ks = np.zeros_like(v), np.full_like(vs, 127)
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    table = torch.arange(n, dtype=torch.int32, device="cuda")[:, None].contiguous()
    q = torch.ones((n, dim), device="cuda")
    out = torch.zeros_like(q)
    starts, lens = torch.arange(n + 1, dtype=torch.int32, device="cuda"), torch.ones(n, dtype=torch.int32, device="cuda")
    hip.PagedAttention(out, q, PagedKVCache(dev(k), dev(v), table, dev(ks), dev(vs)), starts, lens, 1.0)
    want = mx.values(mx.unpack(v[:, 0, 0]), vs[:, 0, 0])
    assert np.array_equal(out.cpu().numpy().astype(np.float64), want)


def test_results_do_not_depend_on_the_batch_or_the_stream(hip):
    import torch
    rng = np.random.default_rng(12)
    contexts, news = [900, 30, 2100, 64], [1, 5, 40, 1]
    c = FourBits(torch, rng, contexts, 16, 2, 128)
    q = torch.from_numpy(rng.standard_normal((sum(news), 8 * 128)).astype(np.float32)).cuda()
    whole = run(hip, torch, c, q, news, contexts, 0.1)
    again = run(hip, torch, c, q, news, contexts, 0.1)
    assert torch.equal(whole, again)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(hip, torch, c, q, news, contexts, 0.1)
    side.synchronize()
    assert torch.equal(whole, other)


def test_a_captured_call_serves_other_lengths(hip):
    import torch
    rng = np.random.default_rng(13)
    heads, kv, dim = 8, 2, 128
    c = FourBits(torch, rng, [1500, 1500, 1500], 16, kv, dim, "head")
    q = torch.from_numpy(rng.standard_normal((24, heads * dim)).astype(np.float32)).cuda()
    starts, lens = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    cache = c.cache()
    with torch.cuda.stream(side):
        call = lambda: hip.PagedAttention(out, q, cache, starts, lens, 0.1, window=700, first=4)  # noqa: E731
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
        for news, contexts in (([1, 1, 1], [1500, 3, 700]), ([22, 1, 1], [1400, 1200, 1]), ([0, 24, 0], [0, 900, 5]), ([1, 1, 1], [1500, 3, 700])):
            starts.copy_(starts_of(news, torch))
            lens.copy_(torch.tensor(contexts, dtype=torch.int32, device="cuda"))
            out.fill_(7.5)
            graph.replay()
            side.synchronize()
            rows = sum(news)
            check(out[:rows], c, q[:rows], news, contexts, heads, dim, 0.1, 700, 4)
            assert torch.all(out[rows:] == 7.5)
