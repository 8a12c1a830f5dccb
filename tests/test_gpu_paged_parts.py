"""GPU: every 16-bit part of what the attention over pages multiplies is there, for every dimension and key by itself.

Queries and keys have one dimension each that is not zero, so a score is one exact product, and a result's element is one weight (or one value).
Bounds: the exponent's argument rounds twice relative to the score and once to its own size, the exponential once, twice for the sum: 2^-23 (2 |s| + 4);
an fp16 cache's queries are held in 22 bits, 2^-21 |s| for a weight and its sum; weights and their sum 2^-20.  A part that is lost changes what it belongs
to by 2^-9 (second) or 2^-17 (third) on average."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def attend(hip, torch, q, k, v, news, scale):
    """all sequences over the same pages of 16; k, v [positions, kv heads, dim], every new token behind all of them"""
    from tensorsharp_amd import PagedKVCache
    n, kv, dim = k.shape
    pages = -(-(n + max(news)) // 16)
    put = [torch.zeros((pages * 16, kv, dim), dtype=t.dtype, device="cuda") for t in (k, v)]
    for to, t in zip(put, (k, v)):
        to[:n] = t
    put = [t.view(pages, 16, kv, dim).flip(0).contiguous() for t in put]
    table = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device="cuda").expand(len(news), -1).contiguous()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out = torch.full_like(q, 7.5)
    hip.PagedAttention(out, q, PagedKVCache(*put, table), i32([0] + list(np.cumsum(news))), i32([n + m for m in news]), scale)
    return out


def weights(scores):
    w = np.exp(scores - scores.max(-1, keepdims=True))
    return w / w.sum(-1, keepdims=True)


def room(scores, dtype):
    s = np.abs(scores).max()
    return 2.0 ** -23 * (2 * s + 4) + (2.0 ** -21 * s if dtype == "float16" else 0.0) + 2.0 ** -20


SHAPES = pytest.mark.parametrize("dim,news", [(d, n) for d in (16, 64, 80, 96, 128, 160, 192, 256) for n in ([1], [4] * 8, [130], [33, 3])])
TYPES = pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])


@TYPES
@SHAPES
@pytest.mark.parametrize("low,high,scale", [(1.0, 1.03125, 256.0), (0.0, 4.0, 1.0), (-3.0, 0.0, -1.0)])
def test_parts_of_queries_and_weights(hip, dtype, dim, news, low, high, scale):
    """keys and values are the unit vectors: a row's result is the softmax of its query's elements"""
    import torch
    rng = np.random.default_rng(dim + len(news))
    one = torch.eye(dim, device="cuda").to(getattr(torch, dtype))[:, None].expand(dim, 2, dim)
    q = rng.uniform(low, high, (sum(news), 2, dim)).astype(np.float32)
    got = attend(hip, torch, torch.from_numpy(q.reshape(sum(news), -1)).cuda(), one, one, news, scale)
    scores = scale * q.astype(np.float64)
    last = np.concatenate([np.arange(1, n + 1) for n in news])                    # keys behind the unit vectors, of score 0
    w = np.exp(scores - np.maximum(scores.max(-1, keepdims=True), 0.0))
    total = w.sum(-1, keepdims=True) + last[:, None, None] * np.exp(-np.maximum(scores.max(-1, keepdims=True), 0.0))
    ref = w / total
    d = np.abs(got.double().cpu().numpy().reshape(ref.shape) - ref)
    assert np.all(d <= room(scores, dtype) * ref), float((d / ref).max())


@SHAPES
def test_parts_of_keys(hip, dim, news):
    """an fp32 cache (keys of 16 bits are one part): row r has dimension r of 40 keys alone for its scores"""
    import torch
    rng = np.random.default_rng(dim)
    rows = sum(news)
    for shift in range(0, dim, max(1, rows)):                       # every dimension's turn
        k = rng.uniform(1.0, 1.03125, (min(dim, 40), 2, dim)).astype(np.float32)
        v = np.broadcast_to(np.eye(dim, dtype=np.float32)[:len(k), None], k.shape)
        q = np.zeros((rows, 2, dim), dtype=np.float32)
        at = (np.arange(rows) + shift) % dim
        q[np.arange(rows), :, at] = 1.0
        got = attend(hip, torch, torch.from_numpy(q.reshape(rows, -1)).cuda(), torch.from_numpy(k).cuda(), torch.from_numpy(v.copy()).cuda(), news, 256.0)
        scores = 256.0 * k.astype(np.float64)[:, :, at].transpose(2, 1, 0)
        ref = weights(scores)                                       # (keys of score 0 are 256 below: nothing in 64 bits)
        d = np.abs(got.double().cpu().numpy().reshape(rows, 2, dim)[..., :len(k)] - ref)
        assert np.all(d <= room(scores, "float32") * ref), (shift, float((d / ref).max()))


@TYPES
@SHAPES
def test_parts_of_values(hip, dtype, dim, news):
    """each row takes one key's value, the others being 200 below: six products and as many roundings, and those of the division"""
    import torch
    rng = np.random.default_rng(dim)
    rows, keys = sum(news), dim
    one = torch.eye(dim, device="cuda").to(getattr(torch, dtype))[:, None].expand(dim, 2, dim)
    v = torch.from_numpy(rng.uniform(1.0, 2.0, (keys, 2, dim)).astype(np.float32)).cuda().to(getattr(torch, dtype))
    q = np.zeros((rows, 2, dim), dtype=np.float32)
    at = (np.arange(rows) * 7) % keys
    q[np.arange(rows), :, at] = 1.0
    got = attend(hip, torch, torch.from_numpy(q.reshape(rows, -1)).cuda(), one, v, news, 200.0).double().view(rows, 2, dim)
    ref = v.double()[torch.from_numpy(at).cuda()]
    assert bool(((got - ref).abs() <= 2.0 ** -20 * ref).all()), float(((got - ref).abs() / ref).max())
