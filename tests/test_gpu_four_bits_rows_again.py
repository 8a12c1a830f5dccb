"""GPU: attention over a cache in four bits where some rows of a tile have NaN or infinities and others have not, the result in the query's place or not.

Of 17 to 32 rows that share a KV head 16 are summed at a time; those with NaN in their sums are done again, each over its own keys.

Bounds.  Rows are held as test_gpu_attention_four_bits.py derives it; one that is done again adds its n keys one after the other, each addition
rounded, which is n 2^-24 of sum p |v| more at worst.  The two places of the result differ in nothing, so these are equal bit for bit."""
import numpy as np
import pytest

from attention_oracle import FourBits, attend
from test_gpu_attention_four_bits import starts_of

pytestmark = pytest.mark.gpu

CASES = [
    # heads, kv heads, dim, new tokens, contexts (of 2000 positions and more the keys are cut)
    (16, 1, 128, [2], [60]),
    (8, 1, 128, [3], [200]),
    (20, 4, 64, [5, 4], [130, 90]),
    (32, 2, 96, [2, 1, 2], [70, 300, 33]),
    (24, 1, 256, [1], [150]),
    (9, 3, 192, [10], [64]),
    (16, 1, 128, [2], [7000]),
    (8, 1, 64, [3, 4], [2500, 6000]),
    (64, 2, 128, [1, 1, 1], [5000, 3001, 40]),
]


@pytest.mark.parametrize("kind", ["query of the last token", "query of the first token", "infinite query", "last key", "last value"])
@pytest.mark.parametrize("heads,kv,dim,news,contexts", CASES)
def test_rows_beside_rows_that_are_done_again(hip, heads, kv, dim, news, contexts, kind):
    import torch
    rng = np.random.default_rng(heads * dim + len(kind))
    group, rows = heads // kv, sum(news)
    assert all(16 < n * group <= 32 for n in news if n > 1 or group > 16)

    def make(i, s, n):
        x = rng.standard_normal((n, kv, dim))
        if kind == ("last key", "last value")[i]:
            x[n - 1, kv - 1, 5] = np.nan
        return x
    c = FourBits(torch, rng, contexts, 16, kv, dim, make=make)
    clean = rng.standard_normal((rows, heads, dim)).astype(np.float32)
    q, whole = clean.copy(), np.zeros((rows, heads), dtype=bool)     # whole: rows that are NaN in all dimensions
    dims = np.zeros((rows, heads, dim), dtype=bool)                  # dimensions that are NaN
    at = 0
    for n in news:
        if "query" in kind:
            row, head = (at, heads - group) if "first" in kind else (at + n - 1, heads - 1)
            q[row, head, dim - 3] = np.inf if "infinite" in kind else np.nan
            whole[row, head] = "infinite" not in kind
        elif kind == "last key":
            whole[at + n - 1, heads - group:] = True
        else:
            dims[at + n - 1, heads - group:, :32] = True
        at += n
    lens = torch.tensor(contexts, dtype=torch.int32, device="cuda")
    qd = torch.from_numpy(q.reshape(rows, -1)).cuda()
    for window, first in ((0, 0), (40, 6)):
        out = torch.full_like(qd, 7.5)
        hip.PagedAttention(out, qd, c.cache(), starts_of(news, torch), lens, 0.1, window=window, first=first)
        place = qd.clone()
        hip.PagedAttention(place, place, c.cache(), starts_of(news, torch), lens, 0.1, window=window, first=first)
        got, same = (t.cpu().numpy().reshape(rows, heads, dim).astype(np.float64) for t in (out, place))
        assert np.array_equal(got, same, equal_nan=True)
        at = 0
        for s, (n, ctx) in enumerate(zip(news, contexts)):
            k, v = (np.nan_to_num(t) for t in c.rows(s, contexts))
            x, y = clean[at:at + n].astype(np.float64), got[at:at + n]
            ref, size = attend(x, k, v, np.arange(ctx - n, ctx), 0.1, window, first)
            nan = whole[at:at + n, :, None] | dims[at:at + n]
            if "infinite" in kind:                                   # (scores of either infinity or NaN: what it gives is not said)
                skip = np.zeros((n, heads, 1), dtype=bool)
                skip[n - 1, heads - 1] = True
            else:
                skip = nan
                assert np.all(np.isnan(y[np.broadcast_to(nan, y.shape)]))
            e = np.zeros((n, heads, 1))
            for h in range(heads):
                keys = np.abs(k[:, h // group])
                most = 0.1 * (np.abs(x[:, h]) @ keys.T).max(1)
                block = np.abs(x[:, h]).reshape(n, -1, 32).max(-1)
                e[:, h, 0] = most * (dim + 12) * 2.0 ** -24 + 4 * 2.0 ** -24
                e[:, h, 0] += 0.1 * 15.0 ** -5 * (block @ keys.reshape(len(keys), -1, 32).sum(-1).T).max(1)
            bound = (2 * e + 2.0 ** -20 + min(ctx, window + first if window else ctx) * 2.0 ** -24) * size
            assert np.all((np.abs(y - ref) <= bound) | skip), (s, float(np.nanmax(np.where(skip, 0.0, np.abs(y - ref) / size))))
            at += n
