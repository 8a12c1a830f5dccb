"""New keys and values into a cache in four bits, against 64 bits.

Values are stored as they come: codes and scales are equal.  Keys are normed and turned in 64 bits and rounded to 32 once, so that a key's code or scale
may be that of a value 2^-24 of its own away (of a turned pair's length; 1 % more for what 64 bits leave) where a border lies between them.  A query is 6e-7
of its pair's length off, 7e-7 of it and of each value more with a norm (test_gpu_rope.py)."""
import numpy as np
import pytest

import mx4_oracle as mx
import paged_oracle as po
from test_gpu_rope import NORM, TURN, description, layout, lengths

pytestmark = pytest.mark.gpu


def four_bits(torch, pages, page, kv, dim, order, gap=0):
    """tensors of codes and scales, heads before or behind tokens, with something in them that no store leaves there"""
    def one(cols, gap):
        shape = (pages, page, kv, cols + gap) if order == "token" else (pages, kv, page, cols + gap)
        t = torch.full(shape, 0xEE, dtype=torch.uint8, device="cuda")[..., :cols]
        return t if order == "token" else t.transpose(1, 2)
    return [one(dim // 2, 16 * gap) for _ in range(2)] + [one(dim // 32, 3 * gap) for _ in range(2)]


@pytest.mark.parametrize("heads,kv,dim,dims,mode,scaling,normed,page,order,gap", [
    (32, 8, 128, 128, 2, "none", True, 16, "token", 0), (8, 8, 64, 32, 0, "yarn", False, 5, "head", 1), (6, 2, 96, 96, 2, "factors", True, 1, "token", 0),
    (5, 1, 256, 64, 0, "linear", True, 64, "head", 0), (7, 7, 32, 32, 2, "none", False, 100, "head", 1), (12, 4, 160, 56, 2, "yarn_part", True, 24, "token", 1),
    (40, 8, 192, 192, 0, "none", False, 32, "token", 0), (9, 3, 224, 88, 0, "yarn", True, 16, "token", 0), (4, 4, 32, 8, 0, "linear", True, 7, "head", 0),
    (1, 1, 128, 4, 2, "none", True, 3, "token", 0)])
def test_store(hip, heads, kv, dim, dims, mode, scaling, normed, page, order, gap):
    import torch
    from tensorsharp_amd import PagedKVCache
    rng = np.random.default_rng(dim + page)
    contexts, news = [70, 1, 33, 9, 201], [1, 1, 33, 0, 120]
    table = po.Cache(torch, rng, contexts, page, 1, 16, torch.float16).table
    parts4 = four_bits(torch, int(table.max()) + 2, page, kv, dim, order, gap)
    cache = PagedKVCache(*parts4[:2], torch.from_numpy(table).cuda(), *parts4[2:])
    starts, lens, position = layout(contexts, news, torch)
    rows = sum(news)
    x = rng.standard_normal((rows + 3, (heads + 2 * kv) * dim)).astype(np.float32)
    x[5, -dim:] = 0.0                                                 # a block of zeros, ties, and one with an infinity
    x[6, -32:] = np.tile(np.float32([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]), 4)
    x[7, -32:] = np.tile(np.float32([-.25, -.75, -1.25, -1.75, -2.5, -3.5, -5.0, 7.0]), 4)
    x[8, -1], x[9, -2], x[10, -32] = np.inf, np.nan, 2.0 ** 127
    qn, kn = ((rng.uniform(0.5, 1.5, dim).astype(np.float32) for _ in range(2)) if normed else (None, None))
    native, kw = description(torch, dims, mode, 500000.0, scaling, rng)
    query = torch.full((rows + 3, heads * dim), 7.5, device="cuda")
    put = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    xd = put(x)
    hip.RoPEStorePaged(query, xd, cache, starts, lens, native, put(qn), put(kn), 1e-5)
    size = abs(po.turns([0], dims, **kw)[0, 0])
    parts = x[:rows].astype(np.float64).reshape(rows, heads + 2 * kv, dim)

    def check(got, part, weight, stored=None):
        y = po.norm(part, weight, 1e-5)
        ref = po.rope(y, position, dims, mode, **kw)
        room = (TURN + (NORM if normed else 0)) * size * lengths(y, dims, mode) + (NORM if normed else 0) * np.abs(y)
        if stored is None:
            assert np.all(np.abs(got - ref) <= room)
        else:
            room = 1.01 * 2.0 ** -24 * np.maximum(size * lengths(y, dims, mode), np.abs(y))
            assert mx.holds(*stored, ref, room.reshape(*room.shape[:-1], -1, 32).max(-1))
    check(query.cpu().numpy()[:rows].reshape(rows, heads, dim), parts[:, :heads], qn)
    assert torch.all(query[rows:] == 7.5)
    where = (np.concatenate([table[s, np.arange(a - n, a) // page] for s, (a, n) in enumerate(zip(contexts, news))]), position % page)
    k, v, ks, vs = (t.cpu().numpy() for t in parts4)
    check(None, parts[:, heads:heads + kv], kn, (k[where], ks[where]))
    values = parts[:, heads + kv:]
    e = mx.scales(values)
    assert np.array_equal(vs[where], e)
    fine = np.repeat(e != 255, 32, axis=-1)
    assert np.array_equal(mx.unpack(v[where])[fine], mx.codes(values, np.where(e == 255, 127, e).astype(np.uint8))[fine])
    assert (e == 255).sum() == 3
    for t in (k, v, ks, vs):                                          # nothing else was written
        t[where] = 0xEE
        assert (t == 0xEE).all()
    # queries in place, and rotation by positions of the caller's
    hip.RoPEStorePaged(xd[:, :heads * dim], xd, cache, starts, lens, native, put(qn), put(kn), 1e-5)
    assert torch.equal(xd[:rows, :heads * dim], query[:rows])
    other = torch.from_numpy(np.concatenate([position + 1000, [0, 0, 0]]).astype(np.int32)).cuda()
    hip.RoPEStorePaged(query, put(x), cache, starts, lens, native, put(qn), put(kn), 1e-5, positions=other)
    position = position + 1000
    check(query.cpu().numpy()[:rows].reshape(rows, heads, dim), parts[:, :heads], qn)
    k, ks = parts4[0].cpu().numpy(), parts4[2].cpu().numpy()
    check(None, parts[:, heads:heads + kv], kn, (k[where], ks[where]))


def test_store_leaves_out_what_has_no_place(hip):
    import torch
    from tensorsharp_amd import PagedKVCache, RotaryPositions
    kv, dim, page = 2, 64, 4
    k, v, ks, vs = (t.zero_() for t in four_bits(torch, 3, page, kv, dim, "token"))
    table = torch.tensor([[1, 5, -2], [2, 0, -1], [-2 ** 31, 2 ** 31 - 1, 3]], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 12, 14, 20], dtype=torch.int32, device="cuda")
    lens = torch.tensor([12, 1, 15], dtype=torch.int32, device="cuda")
    x = torch.randn((20, (2 + 2 * kv) * dim), device="cuda")
    query = torch.zeros((20, 2 * dim), device="cuda")
    hip.RoPEStorePaged(query, x, PagedKVCache(k, v, table, ks, vs), starts, lens, RotaryPositions(dim))
    assert torch.all(query.abs().sum(1) > 0)
    for scales in (ks, vs):
        assert (scales > 0).all(3).all(2).tolist() == [[False] * 4, [True] * 4, [True, False, False, False]]
        assert (scales > 0).any(3).any(2).tolist() == [[False] * 4, [True] * 4, [True, False, False, False]]
