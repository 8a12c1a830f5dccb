"""GPU: windows with first positions over caches of 16 and 32 bits where some rows have NaN in their query or see keys or values with NaN (in the first positions, in
the window, or between them, where nobody looks), the result in the query's place or not.

Bounds as test_gpu_paged_attention.py derives them, and n 2^-24 of sum p |v| for the n keys that a row which is done again adds one after the other."""
import numpy as np
import pytest

import paged_oracle as po
from attention_oracle import attend
from test_gpu_attention_four_bits import starts_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["query", "keys", "values"])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("heads,kv,dim,news,contexts", [(16, 1, 64, [2, 1], [90, 40]), (20, 4, 128, [5, 4], [300, 200]), (8, 2, 256, [3], [150]), (6, 2, 96, [50, 1], [180, 77]),
                                                        (16, 1, 128, [2, 1], [2500, 400])])
def test_rows_with_and_without_nan(hip, heads, kv, dim, news, contexts, dtype, kind):
    import torch
    from tensorsharp_amd import PagedKVCache
    rng = np.random.default_rng(heads * dim + len(kind))
    c = po.Cache(torch, rng, contexts, 16, kv, dim, getattr(torch, dtype))
    group, rows = heads // kv, sum(news)
    bad = [[3, n // 2, n - 1] for n in contexts]                     # positions of keys or values with NaN in the last KV head
    if kind != "query":
        t = c.k if kind == "keys" else c.v
        for s, at in enumerate(bad):
            for p in at:
                t[int(c.table[s, p // 16]), p % 16, kv - 1, 5] = float("nan")
    clean = rng.standard_normal((rows, heads, dim)).astype(np.float32)
    q = clean.copy()
    lost = np.zeros((rows, heads), dtype=bool)
    if kind == "query":
        at = 0
        for n in news:
            q[at + n - 1, heads - 1, dim - 1] = np.nan
            lost[at + n - 1, heads - 1] = True
            at += n
    qd = torch.from_numpy(q.reshape(rows, -1)).cuda()
    lens, starts = torch.tensor(contexts, dtype=torch.int32, device="cuda"), starts_of(news, torch)
    cache = PagedKVCache(c.k, c.v, c.table_dev)
    for window, first in ((20, 2), (20, 4), (7, 40), (2 ** 31 - 1, 4)):
        out = torch.full_like(qd, 7.5)
        hip.PagedAttention(out, qd, cache, starts, lens, 0.1, window=window, first=first)
        place = qd.clone()
        hip.PagedAttention(place, place, cache, starts, lens, 0.1, window=window, first=first)
        got, same = (t.cpu().numpy().reshape(rows, heads, dim).astype(np.float64) for t in (out, place))
        assert np.array_equal(got, same, equal_nan=True)
        at = 0
        for s, (n, ctx) in enumerate(zip(news, contexts)):
            k, v = (np.nan_to_num(t) for t in c.rows(s, contexts))
            p = np.arange(ctx - n, ctx)
            x, y = clean[at:at + n].astype(np.float64), got[at:at + n]
            ref, size = attend(x, k, v, p, 0.1, window, first)
            sees = np.array([any(b <= i and (b > i - window or b < first) for b in bad[s]) for i in p])
            nan = np.zeros(y.shape, dtype=bool)
            if kind == "query":
                nan[lost[at:at + n]] = True
            elif kind == "keys":
                nan[sees, heads - group:] = True
            else:
                nan[sees, heads - group:, 5] = True
            assert np.array_equal(np.isnan(y), nan)
            e = np.zeros((n, heads, 1))
            for h in range(heads):
                most = 0.1 * (np.abs(x[:, h]) @ np.abs(k[:, h // group]).T).max(1)
                e[:, h, 0] = most * ((dim + 12) * 2.0 ** -24 + 2.0 ** -21) + 4 * 2.0 ** -24
            bound = (2 * e + 2.0 ** -20 + min(ctx, window + first) * 2.0 ** -24) * size
            assert np.all((np.abs(y - ref) <= bound) | nan), (s, window, first)
            at += n
