"""GPU: powers that no store writes (2^-127, 2^126, 2^127) but that a cache in four bits may hold: keys, values and copies of them are what their codes stand for.

Bounds.  A single key's result is its value; what is beyond fp32's largest is infinite there.  Means of two or four values of one weight are rounded once
for each key at most: 8 x 2^-24.  Scores are single products of powers of two and codes, exact; weights and their sum round 8 x 2^-24."""
import numpy as np
import pytest

import mx4_oracle as mx

pytestmark = pytest.mark.gpu
POWERS = [0, 253, 254]


def cache_of(torch, k, ks, v, vs):
    """one page of one head for each sequence; codes [seqs, keys, 32] and powers [seqs, keys]"""
    from tensorsharp_amd import PagedKVCache
    put = lambda c: torch.from_numpy(mx.pack(c.astype(np.uint8))[:, :, None].copy()).cuda()  # noqa: E731
    power = lambda e: torch.from_numpy(e.astype(np.uint8)[:, :, None, None].copy()).cuda()  # noqa: E731
    table = torch.arange(len(k), dtype=torch.int32, device="cuda")[:, None].contiguous()
    return PagedKVCache(put(k), put(v), table, power(ks), power(vs))


def attend(hip, torch, cache, q, keys, scale, rows=1):
    seqs = len(q) // rows
    out = torch.full_like(q, 7.5)
    starts = torch.arange(0, seqs * rows + 1, rows, dtype=torch.int32, device="cuda")
    lens = torch.full((seqs,), keys, dtype=torch.int32, device="cuda")
    hip.PagedAttention(out, q, cache, starts, lens, scale)
    return out.cpu().numpy().astype(np.float64)


@pytest.mark.parametrize("e", POWERS)
def test_single_values(hip, e):
    import torch
    v = np.tile(np.arange(32) % 16, (2, 1, 1))
    zero = np.zeros_like(v)
    got = attend(hip, torch, cache_of(torch, zero, np.full((2, 1), 127), v, np.full((2, 1), e)), torch.ones((2, 32), device="cuda"), 1, 1.0)
    with np.errstate(over="ignore"):
        want = mx.values(v[:, 0], np.full((2, 1), e, dtype=np.uint8)).astype(np.float32).astype(np.float64)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("heads", [1, 40])
@pytest.mark.parametrize("keys", [2, 4])
@pytest.mark.parametrize("e", POWERS)
def test_means_of_values(hip, e, keys, heads):
    """of which fp32 holds the mean, whether it holds the values or not"""
    import torch
    v = np.zeros((3, keys, 32), dtype=np.int64)
    v[0, 0] = np.arange(32) % 16                                     # one value, the others 0
    v[1] = 3                                                         # alike
    v[2, 0], v[2, 1] = 7, 15                                         # the largest and its opposite
    if e == 254:
        v[0, 0] %= 6 if keys == 4 else 4
        v[1] = 1
    zero = np.zeros_like(v)
    cache = cache_of(torch, zero, np.full((3, keys), 127), v, np.full((3, keys), e))
    want = mx.values(v, np.full((3, keys, 1), e, dtype=np.uint8)).mean(1)
    assert np.all(np.abs(want) < 2.0 ** 128)
    q = torch.ones((3, 32 * heads), device="cuda")
    got = attend(hip, torch, cache, q, keys, 1.0).reshape(3, heads, 32)
    # (the last power of all, 2^-149, where results are smaller than fp32's normal numbers)
    assert np.all(np.abs(got - want[:, None]) <= 8 * 2.0 ** -24 * np.abs(want[:, None]) + 4 * 2.0 ** -149)


@pytest.mark.parametrize("heads", [1, 40])
@pytest.mark.parametrize("e", POWERS)
def test_means_over_pieces_of_keys(hip, e, heads):
    """4096 keys of one weight, cut into pieces.  A block of 64 keys rounds what was summed before it and its own weights, 4 x 2^-24 of sum p |v|, the join 16 x 2^-24."""
    import torch
    keys = 4096
    v = np.zeros((3, keys, 32), dtype=np.int64)
    v[0, 77] = np.arange(32) % 16                                    # one value, the others 0
    v[1] = 3 if e < 254 else 1                                       # alike
    v[2, 0::2], v[2, 1::2] = 7, 15                                   # the largest and its opposite
    cache = cache_of(torch, np.zeros_like(v), np.full((3, keys), 127), v, np.full((3, keys), e))
    values = mx.values(v, np.full((3, keys, 1), e, dtype=np.uint8))
    got = attend(hip, torch, cache, torch.ones((3, 32 * heads), device="cuda"), keys, 1.0).reshape(3, heads, 32)
    bound = (4 * keys / 64 + 16) * 2.0 ** -24 * np.abs(values).mean(1) + 2.0 ** -140
    assert np.all(np.abs(got - values.mean(1)[:, None]) <= bound[:, None])


@pytest.mark.parametrize("heads", [1, 40])
@pytest.mark.parametrize("e", POWERS)
def test_keys(hip, e, heads):
    """the first key is zero and has the value 1, the second a code in one dimension and the value -1"""
    import torch
    codes = np.arange(16)
    k = np.zeros((16, 2, 32), dtype=np.int64)
    k[:, 1, 9] = codes
    v = np.full((16, 2, 32), 2)
    v[:, 1] = 10
    ks = np.full((16, 2), e)
    cache = cache_of(torch, k, ks, v, np.full((16, 2), 127))
    q, scale = (2.0 ** 100, 2.0 ** 27) if e == 0 else (2.0 ** -120, 2.0 ** (246 - e - 1) / 2.0)
    s = mx.values(codes[:, None] * np.ones((1, 32), dtype=np.int64), np.full((16, 1), e, dtype=np.uint8))[:, 0] * q * scale
    assert 0.5 < np.abs(s).max() < 2.0 ** 8
    want = np.tanh(-s / 2.0)
    got = attend(hip, torch, cache, torch.full((16, 32 * heads), q, device="cuda"), 2, scale)
    assert np.all(np.abs(got - want[:, None]) <= 2.0 ** -20 + 2 * np.abs(s[:, None]) * 8 * 2.0 ** -24)


@pytest.mark.parametrize("e", POWERS)
def test_copies(hip, e):
    import torch
    from tensorsharp_amd import PagedKVCache
    v = np.tile(np.arange(32) % 16, (2, 3, 1))
    four = cache_of(torch, v, np.full((2, 3), e), v, np.full((2, 3), e))
    moves = torch.tensor([[0, 1], [1, 0]], dtype=torch.int32, device="cuda")
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        wide = PagedKVCache(torch.zeros((2, 3, 1, 32), dtype=dtype, device="cuda"), torch.zeros((2, 3, 1, 32), dtype=dtype, device="cuda"), four.page_table)
        hip.CopyPages(wide, four, moves)
        with np.errstate(over="ignore"):
            want = torch.from_numpy(mx.values(v, np.full((2, 3, 1), e, dtype=np.uint8)).astype(np.float32)).to(dtype)
        assert torch.equal(wide.k.cpu()[:, :, 0], want) and torch.equal(wide.v.cpu()[:, :, 0], want)
