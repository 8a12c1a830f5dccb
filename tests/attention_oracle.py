"""Attention over keys of which a token sees a window and the first ones, in 64 bits, and caches for it, for the tests."""
import numpy as np

import mx4_oracle as mx
import paged_oracle as po


def attend(q, k, v, position, scale, window=0, first=0, sinks=None, present=None):
    """One sequence: q [rows, heads, dim] at positions `position`, k / v [keys, kv heads, dim] -> result, sum_j p_j |v_j| [rows, heads, dim]"""
    q, k, v = (np.asarray(t, dtype=np.float64) for t in (q, k, v))
    rows, heads, dim = q.shape
    group = heads // k.shape[1]
    j = np.arange(len(k))
    position = np.asarray(position)[:, None]
    seen = j[None, :] <= position
    if window:
        seen &= (j[None, :] > position - window) | (j[None, :] < first)
    if present is not None:
        seen &= present[None, :]
    out, size = np.zeros_like(q), np.zeros_like(q)
    for h in range(heads):
        s = np.where(seen, scale * (q[:, h] @ k[:, h // group].T), -np.inf)
        m = s.max(1, initial=-np.inf, keepdims=True)
        if sinks is not None:
            m = np.maximum(m, float(sinks[h]))
        some = np.isfinite(m[:, 0])
        w = np.exp(s[some] - m[some])
        total = w.sum(1, keepdims=True) + (0.0 if sinks is None else np.exp(float(sinks[h]) - m[some]))
        out[some, h] = w @ v[:, h // group] / total
        size[some, h] = w @ np.abs(v[:, h // group]) / total
    return out, size


class FourBits:
    """Pages of codes and scales for sequences of `contexts` tokens, shuffled over memory, heads before or behind tokens; as in paged_oracle.Cache
    what lies behind a sequence's last token is NaN."""

    def __init__(self, torch, rng, contexts, page, kv_heads, dim, order="token", make=None):
        self.page, self.contexts, self.torch = page, list(contexts), torch
        plan = po.Cache(torch, rng, contexts, page, 1, 16, torch.float16, fill=False)
        self.table, self.table_dev = plan.table, plan.table_dev
        pages = plan.k.shape[0]
        self.codes = [rng.integers(0, 256, (pages, page, kv_heads, dim // 2)).astype(np.uint8) for _ in range(2)]
        self.scales = [np.full((pages, page, kv_heads, dim // 32), 255, dtype=np.uint8) for _ in range(2)]
        for s, c in enumerate(contexts):
            p = np.arange(c)
            where = (self.table[s, p // page], p % page)
            for i in range(2):
                x = rng.standard_normal((c, kv_heads, dim)) if make is None else make(i, s, c)
                e = mx.scales(x)
                self.scales[i][where], self.codes[i][where] = e, mx.pack(mx.codes(x, np.where(e == 255, 127, e).astype(np.uint8)))
        put = lambda a: torch.from_numpy(a if order == "token" else np.ascontiguousarray(a.transpose(0, 2, 1, 3))).cuda()  # noqa: E731
        self.device = [put(t) if order == "token" else put(t).transpose(1, 2) for t in (*self.codes, *self.scales)]

    def cache(self, table=None):
        from tensorsharp_amd import PagedKVCache
        k, v, ks, vs = self.device
        return PagedKVCache(k, v, self.table_dev if table is None else table, ks, vs)

    def rows(self, s, contexts=None):
        p = np.arange((contexts or self.contexts)[s])
        where = (self.table[s, p // self.page], p % self.page)
        return tuple(mx.values(mx.unpack(c[where]), e[where]) for c, e in zip(self.codes, self.scales))
