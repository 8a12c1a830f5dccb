"""GPU: rotary positions alone, and with the norm and the store into a paged cache, against their definition in 64 bits.

Bound of a turned pair (a, b), relative to its length: the angle in revolutions is rounded to 32 bits once (2^-26 of a revolution at
most, 9.4e-8 radians), sine and cosine are within two units of 2^-24 (1.2e-7 each, 1.7e-7 together), two products and a sum round
three times (1.8e-7), size once more: 5e-7, held to 6e-7.  The norm adds what a sum of squares (eight roundings on the way), a
division, a root and two products round: 12 x 2^-24 = 7e-7.  A store in 16 bits adds half a step of its type."""
import numpy as np
import pytest

import paged_oracle as po

gpu = pytest.mark.gpu
TURN, NORM = 6e-7, 7e-7
SCALINGS = {"none": {}, "linear": {"freq_scale": 1 / 3}, "yarn": {"freq_scale": 0.0625, "ext_factor": 1.0, "original_context": 8192},
            "yarn_part": {"freq_scale": 0.25, "ext_factor": 0.7, "attn_factor": 1.1, "beta_fast": 16.0, "beta_slow": 2.0, "original_context": 4096}}


def lengths(x, dims, mode):
    """of the pair that each dimension is in (of a dimension that is not turned: 0)"""
    out = np.zeros(x.shape)
    a, b = (slice(0, dims // 2), slice(dims // 2, dims)) if mode == 2 else (slice(0, dims, 2), slice(1, dims, 2))
    out[..., a] = out[..., b] = np.hypot(x[..., a], x[..., b])
    return out


def description(torch, dims, mode, base, scaling, rng):
    from tensorsharp_amd import RotaryPositions
    kw = dict(SCALINGS[scaling]) if scaling != "factors" else {}
    factors = rng.uniform(1, 8, dims // 2).astype(np.float32) if scaling == "factors" else None
    native = RotaryPositions(dims, mode=mode, base=base, freq_factors=None if factors is None else torch.from_numpy(factors).cuda(), **kw)
    return native, dict(kw, base=base, freq_factors=factors)


@gpu
@pytest.mark.parametrize("tokens,heads,dim,dims,mode,base,scaling,far", [
    (1, 1, 128, 128, 2, 10000.0, "none", 1), (1, 32, 128, 128, 0, 500000.0, "factors", 8192), (5, 3, 64, 32, 2, 10000.0, "linear", 300),
    (33, 7, 80, 20, 0, 10000.0, "yarn", 131072), (257, 8, 96, 96, 2, 1e6, "yarn_part", 4096), (19, 5, 256, 256, 2, 1e6, "none", 2000000000),
    (3, 2, 4, 4, 0, 10000.0, "none", 100), (2100, 2, 36, 8, 2, 10000.0, "none", 5000), (64, 40, 192, 96, 0, 500000.0, "yarn", 100000)])
def test_rope(hip, tokens, heads, dim, dims, mode, base, scaling, far):
    import torch
    rng = np.random.default_rng(tokens + dim)
    x = rng.standard_normal((tokens, heads, dim)).astype(np.float32)
    pos = rng.integers(0, far, tokens).astype(np.int32)
    native, kw = description(torch, dims, mode, base, scaling, rng)
    ref = po.rope(x, pos, dims, mode, **kw)
    xd = torch.from_numpy(x).cuda()
    out = torch.full_like(xd, float("nan"))
    hip.RoPE(out, xd, torch.from_numpy(pos).cuda(), native)
    got = out.cpu().numpy()
    size = abs(po.turns([0], dims, **kw)[0, 0])
    assert np.all(np.abs(got - ref) <= TURN * size * lengths(x.astype(np.float64), dims, mode))
    assert np.array_equal(got[..., dims:], x[..., dims:])
    # in place, and as heads before tokens in memory
    hip.RoPE(xd, xd, torch.from_numpy(pos).cuda(), native)
    assert torch.equal(xd, out)
    swapped = torch.from_numpy(np.ascontiguousarray(x.transpose(1, 0, 2))).cuda().transpose(0, 1)
    other = torch.zeros((tokens, heads + 1, dim + 4), device="cuda")[:, 1:, :dim]
    hip.RoPE(other, swapped, torch.from_numpy(pos).cuda(), native)
    assert torch.equal(other, out)


@gpu
def test_rope_of_negative_positions_and_far_ones(hip):
    import torch
    from tensorsharp_amd import RotaryPositions
    pos = np.array([-1, -70000, 2 ** 31 - 1, -2 ** 31, 0], dtype=np.int32)
    x = np.random.default_rng(3).standard_normal((5, 2, 64)).astype(np.float32)
    out = torch.from_numpy(x).cuda()
    hip.RoPE(out, out, torch.from_numpy(pos).cuda(), RotaryPositions(64, mode=2, base=10000.0))
    assert np.all(np.abs(out.cpu().numpy() - po.rope(x, pos, 64)) <= TURN * lengths(x.astype(np.float64), 64, 2))
    assert np.array_equal(out.cpu().numpy()[4], x[4])


def layout(contexts, news, torch):
    starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    position = np.concatenate([np.arange(c - n, c) for c, n in zip(contexts, news)])
    return torch.from_numpy(starts).cuda(), torch.tensor(contexts, dtype=torch.int32, device="cuda"), position


@gpu
@pytest.mark.parametrize("heads,kv,dim,dims,mode,scaling,normed,dtype,page,order", [
    (32, 8, 128, 128, 2, "none", True, "float16", 16, "token"), (8, 8, 64, 32, 0, "yarn", False, "bfloat16", 5, "head"),
    (6, 2, 80, 80, 2, "factors", True, "float32", 1, "token"), (5, 1, 256, 64, 0, "linear", True, "float16", 64, "head"),
    (7, 7, 16, 16, 2, "none", False, "float32", 100, "head"), (12, 4, 112, 56, 2, "yarn_part", True, "bfloat16", 24, "token"),
    (40, 8, 192, 192, 0, "none", False, "float16", 32, "token"), (9, 3, 176, 88, 0, "yarn", True, "bfloat16", 16, "token"),
    (4, 4, 256, 256, 2, "linear", True, "float32", 7, "head"), (8, 2, 32, 32, 0, "none", True, "float16", 16, "token"),
    (6, 1, 16, 8, 2, "factors", False, "bfloat16", 3, "head")])
def test_store(hip, heads, kv, dim, dims, mode, scaling, normed, dtype, page, order):
    import torch
    from tensorsharp_amd import PagedKVCache
    rng = np.random.default_rng(dim + page)
    contexts, news = [70, 1, 33, 9, 201], [1, 1, 33, 0, 120]
    t = getattr(torch, dtype)
    c = po.Cache(torch, rng, contexts, page, kv, dim, t, order)
    before = [a.clone() for a in (c.k, c.v)]
    starts, lens, position = layout(contexts, news, torch)
    rows = sum(news)
    x = rng.standard_normal((rows + 3, (heads + 2 * kv) * dim)).astype(np.float32)
    qn, kn = ((rng.uniform(0.5, 1.5, dim).astype(np.float32) for _ in range(2)) if normed else (None, None))
    native, kw = description(torch, dims, mode, 500000.0, scaling, rng)
    xd = torch.from_numpy(x).cuda()
    query = torch.full((rows + 3, heads * dim), 7.5, device="cuda")
    put = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    cache = PagedKVCache(c.k, c.v, c.table_dev)
    hip.RoPEStorePaged(query, xd, cache, starts, lens, native, put(qn), put(kn), 1e-5)
    size = abs(po.turns([0], dims, **kw)[0, 0])
    parts = x[:rows].reshape(rows, heads + 2 * kv, dim)
    step = {"float32": 0.0, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}[dtype]
    tiny = {"float32": 0.0, "float16": 2.0 ** -25, "bfloat16": 0.0}[dtype]          # half a step of a subnormal

    def check(got, part, weight, rounding):
        y = po.norm(part, weight, 1e-5)
        ref = po.rope(y, position, dims, mode, **kw)
        room = (TURN + (NORM if normed else 0)) * size * lengths(y, dims, mode) + (NORM if normed else 0) * np.abs(y)
        assert np.all(np.abs(got - ref) <= room + rounding * (np.abs(ref) + room) + (tiny if rounding else 0))
    check(query.cpu().numpy()[:rows].reshape(rows, heads, dim), parts[:, :heads], qn, 0.0)
    assert torch.all(query[rows:] == 7.5)                                         # rows of no sequence
    where = (np.concatenate([c.table[s, np.arange(a - n, a) // page] for s, (a, n) in enumerate(zip(contexts, news))]), position % page)
    check(c.k.float().cpu().numpy()[where], parts[:, heads:heads + kv], kn, step)
    assert torch.equal(c.v.cpu()[where], torch.from_numpy(np.ascontiguousarray(parts[:, heads + kv:])).to(t))
    for a, b in zip((c.k, c.v), before):                                          # nothing else was written
        a, b = a.clone(), b.clone()
        a[where] = b[where] = 0
        assert torch.equal(torch.nan_to_num(a.float(), 3.0), torch.nan_to_num(b.float(), 3.0))
    # queries in place, and rotation by positions of the caller's
    hip.RoPEStorePaged(xd[:, :heads * dim], xd, cache, starts, lens, native, put(qn), put(kn), 1e-5)
    assert torch.equal(xd[:rows, :heads * dim], query[:rows])
    other = torch.from_numpy(np.concatenate([position + 1000, [0, 0, 0]]).astype(np.int32)).cuda()
    hip.RoPEStorePaged(query, torch.from_numpy(x).cuda(), cache, starts, lens, native, put(qn), put(kn), 1e-5, positions=other)
    position = position + 1000
    check(query.cpu().numpy()[:rows].reshape(rows, heads, dim), parts[:, :heads], qn, 0.0)


@gpu
def test_store_leaves_out_what_has_no_place(hip):
    """Pages outside the cache, positions beyond the table and before the first: not stored; the queries come all the same."""
    import torch
    from tensorsharp_amd import PagedKVCache, RotaryPositions
    kv, dim, page = 2, 64, 4
    k = torch.zeros((3, page, kv, dim), device="cuda", dtype=torch.float16)
    v = torch.zeros_like(k)
    table = torch.tensor([[1, 5, -2], [2, 0, -1], [-2 ** 31, 2 ** 31 - 1, 3]], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 12, 14, 20], dtype=torch.int32, device="cuda")
    lens = torch.tensor([12, 1, 15], dtype=torch.int32, device="cuda")            # sequence 1: its first token would be at -1
    x = torch.randn((20, (2 + 2 * kv) * dim), device="cuda")
    query = torch.zeros((20, 2 * dim), device="cuda")
    hip.RoPEStorePaged(query, x, PagedKVCache(k, v, table), starts, lens, RotaryPositions(dim))
    assert torch.all(query.abs().sum(1) > 0)
    stored = (v.abs().sum((2, 3)) > 0).cpu().numpy()
    assert stored.tolist() == [[False] * 4, [True] * 4, [True, False, False, False]]
