"""Rotary positions, attention over a paged cache and sampling written out in 64 bits with numpy, for the tests.

`Cache` lays out a paged cache of given lengths; the definitions below are loops over sequences, heads and rows."""
import numpy as np


def turns(positions, dims, base=10000.0, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0, original_context=0,
          freq_factors=None):
    """complex [tokens, dims / 2]: size e^(i theta)"""
    out = np.zeros((len(positions), dims // 2), dtype=np.complex128)
    for i in range(dims // 2):
        w = base ** (-2.0 * i / dims)
        if freq_factors is not None:
            w /= float(freq_factors[i])
        size, kept = attn_factor, 0.0
        if ext_factor:
            pair = lambda beta: dims * np.log(original_context / (2 * np.pi * beta)) / (2 * np.log(base))  # noqa: E731
            low, high = max(0.0, np.floor(pair(beta_fast))), min(dims - 1.0, np.ceil(pair(beta_slow)))
            kept = ext_factor * (1.0 - min(1.0, max(0.0, (i - low) / max(high - low, 0.001))))
            size *= 1.0 + 0.1 * np.log(1.0 / freq_scale)
        w *= freq_scale * (1.0 - kept) + kept
        out[:, i] = size * np.exp(1j * np.asarray(positions, dtype=np.float64) * w)
    return out


def rope(x, positions, dims, mode=2, **scaling):
    """x [tokens, heads, head_dim]"""
    out = np.array(x, dtype=np.float64)
    t = turns(positions, dims, **scaling)[:, None, :]
    a, b = (slice(0, dims // 2), slice(dims // 2, dims)) if mode == 2 else (slice(0, dims, 2), slice(1, dims, 2))
    z = (out[..., a] + 1j * out[..., b]) * t
    out[..., a], out[..., b] = z.real, z.imag
    return out


def norm(x, weight, eps):
    x = np.asarray(x, dtype=np.float64)
    return x if weight is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, dtype=np.float64)


def attend(q, k, v, position, scale, window=0, sinks=None, present=None):
    """One sequence: q [rows, heads, dim] at positions `position`, k / v [keys, kv heads, dim] (present: which of them are there)
    -> (result, sum_j p_j |v_j|) [rows, heads, dim], both 64 bits"""
    q, k, v = (np.asarray(t, dtype=np.float64) for t in (q, k, v))
    rows, heads, dim = q.shape
    group = heads // k.shape[1]
    out, size = np.zeros_like(q), np.zeros_like(q)
    for r in range(rows):
        lo = max(0, position[r] - window + 1) if window else 0
        js = np.arange(lo, min(position[r] + 1, len(k)))
        if present is not None:
            js = js[present[js]]
        if len(js) == 0:
            continue
        for h in range(heads):
            s = scale * (k[js, h // group] @ q[r, h])
            m = max(s.max(), -np.inf if sinks is None else float(sinks[h]))
            w = np.exp(s - m)
            total = w.sum() + (0.0 if sinks is None else np.exp(float(sinks[h]) - m))
            out[r, h] = w @ v[js, h // group] / total
            size[r, h] = w @ np.abs(v[js, h // group]) / total
    return out, size


def sample(logits, u, temperature, top_k=0, top_p=1.0, min_p=0.0):
    """(token, its probability) of one row"""
    x = np.asarray(logits, dtype=np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    if x.max() == -np.inf:
        return -1, 0.0
    if not temperature > 0:
        return int(np.argmax(x)), 1.0
    ids = np.argsort(-x, kind="stable")
    ids = ids[x[ids] > -np.inf]
    if top_k > 0:
        ids = ids[:top_k]
    top, temperature = x.max(), float(np.float32(temperature))
    with np.errstate(invalid="ignore"):
        weight = lambda i: np.where(x[i] == top, 1.0, np.exp((x[i] - top) / temperature))  # noqa: E731
        if np.float32(top_p) < 1:
            cum = np.cumsum(weight(ids))
            ids = ids[:1 + min(len(ids) - 1, int(np.searchsorted(cum, float(np.float32(top_p)) * cum[-1])))]
        stays = weight(ids) >= float(np.float32(min_p))
        stays[0] = True
        ids = ids[stays]
        ids = np.sort(ids)
        cum = np.cumsum(weight(ids))
    at = min(int(np.searchsorted(cum, float(np.float32(u)) * cum[-1], side="right")), len(ids) - 1)
    return int(ids[at]), float(weight(ids[at]) / cum[-1])


class Cache:
    """Pages for sequences of `contexts` tokens, shuffled over memory.  k / v: torch tensors [pages, page, kv heads, dim] on the device
    (heads before tokens in memory where order is "head"); rows(s): the sequence's keys and values as 64-bit numpy arrays.
    What lies behind a sequence's last token is NaN."""

    def __init__(self, torch, rng, contexts, page, kv_heads, dim, dtype, order="token", spare=2, fill=True):
        self.page, self.contexts = page, list(contexts)
        counts = [-(-c // page) for c in contexts]
        pages = sum(counts) + spare
        ids = rng.permutation(pages)
        self.table = np.full((len(contexts), max(counts) + 1), -1, dtype=np.int32)
        shape = (pages, page, kv_heads, dim)
        self.host = [np.full(shape, np.nan, dtype=np.float32) for _ in range(2)]
        at = 0
        for s, (c, n) in enumerate(zip(contexts, counts)):
            self.table[s, :n] = ids[at:at + n]
            at += n
            if fill:
                p = np.arange(c)
                for t in self.host:
                    t[self.table[s, p // page], p % page] = rng.standard_normal((c, kv_heads, dim))
        put = lambda a: torch.from_numpy(a if order == "token" else np.ascontiguousarray(a.transpose(0, 2, 1, 3))).cuda().to(dtype)  # noqa: E731
        self.k, self.v = (put(t) if order == "token" else put(t).transpose(1, 2) for t in self.host)
        self.table_dev = torch.from_numpy(self.table).cuda()
        self.dtype, self.torch = dtype, torch

    def rows(self, s, contexts=None):
        p = np.arange((contexts or self.contexts)[s])
        where = (self.table[s, p // self.page], p % self.page)
        return tuple(t.float().cpu().numpy()[where].astype(np.float64) for t in (self.k, self.v))
