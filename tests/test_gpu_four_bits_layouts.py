"""GPU: caches in four bits whose keys, values and scales lie in memory in different orders, and far apart: what is stored and what attention gives are the same
bits as with everything packed, since the same numbers are computed in the same order."""
import numpy as np
import pytest

from attention_oracle import FourBits
from test_gpu_attention_four_bits import check, starts_of

pytestmark = pytest.mark.gpu


def laid_out(torch, shape, order, gaps=(0, 0, 0, 0)):
    """an empty tensor [pages, tokens, heads, columns] whose dimensions lie in memory in this order (outermost first), with gaps behind each"""
    memory = torch.full([shape[d] + gaps[d] for d in order], 0xEE, dtype=torch.uint8, device="cuda")
    back = [order.index(d) for d in range(4)]
    return memory.permute(back)[tuple(slice(0, n) for n in shape)], memory


LAYOUTS = [
    # k, v, scales of k, scales of v: order of (0 pages, 1 tokens, 2 heads), columns last, and gaps
    ((0, 1, 2, 3), (0, 2, 1, 3), (0, 1, 2, 3), (0, 2, 1, 3), 0), ((0, 2, 1, 3), (0, 1, 2, 3), (0, 1, 2, 3), (0, 1, 2, 3), 1), ((1, 0, 2, 3), (2, 0, 1, 3), (2, 1, 0, 3), (1, 2, 0, 3), 0),
    ((2, 1, 0, 3), (0, 1, 2, 3), (0, 2, 1, 3), (1, 0, 2, 3), 2), ((0, 1, 2, 3), (0, 1, 2, 3), (0, 1, 2, 3), (0, 1, 2, 3), 1)]


@pytest.mark.parametrize("heads,kv,dim,page", [(32, 8, 128, 16), (6, 2, 96, 5), (8, 8, 32, 33), (4, 2, 256, 1), (10, 2, 64, 64)])
@pytest.mark.parametrize("layout", range(len(LAYOUTS)))
def test_orders_in_memory(hip, heads, kv, dim, page, layout):
    import torch
    from tensorsharp_amd import PagedKVCache, RotaryPositions
    rng = np.random.default_rng(dim + layout)
    contexts, news = [700, 40, 1, 260], [1, 40, 1, 7]
    c = FourBits(torch, rng, contexts, page, kv, dim)
    *orders, gap = LAYOUTS[layout]
    gaps = [(gap, gap, gap, 16 * gap)] * 2 + [(gap, 0, gap, gap)] * 2
    there = [laid_out(torch, t.shape, o, g) for t, o, g in zip(c.device, orders, gaps)]
    for (t, _), was in zip(there, c.device):
        t.copy_(was)
    plain, other = c.cache(), PagedKVCache(there[0][0], there[1][0], c.table_dev, there[2][0], there[3][0])
    rows, starts, lens = sum(news), starts_of(news, torch), torch.tensor(contexts, dtype=torch.int32, device="cuda")
    x = torch.from_numpy(rng.standard_normal((rows, (heads + 2 * kv) * dim)).astype(np.float32)).cuda()
    q = [torch.empty((rows, heads * dim), device="cuda") for _ in range(2)]
    for query, cache in zip(q, (plain, other)):
        hip.RoPEStorePaged(query, x, cache, starts, lens, RotaryPositions(dim))
    assert torch.equal(*q)
    for (t, memory), was in zip(there, c.device):
        assert torch.equal(t, was)
        assert int((memory == 0xEE).sum()) >= memory.numel() - t.numel()      # (and not a byte of the gaps)
    for window, first in ((0, 0), (50, 0), (33, 5)):
        out = [torch.empty((rows, heads * dim), device="cuda") for _ in range(2)]
        for o, cache in zip(out, (plain, other)):
            hip.PagedAttention(o, q[0], cache, starts, lens, dim ** -0.5, window=window, first=first)
        assert torch.equal(*out), (window, first)


def test_pages_whose_offsets_pass_32_bits(hip):
    """pages 2^31 bytes apart (and their scales 2^30), as those of a cache are whose layers lie inside a page: the last is 2^33 bytes behind the first"""
    import torch
    from tensorsharp_amd import PagedKVCache, RotaryPositions
    rng = np.random.default_rng(5)
    heads, kv, dim, page, contexts = 8, 2, 128, 64, [129, 200, 30]
    c = FourBits(torch, rng, contexts, page, kv, dim)
    pages = c.codes[0].shape[0]
    assert pages >= 5

    def far(t, apart):
        memory = torch.empty((pages - 1) * apart + t[0].numel(), dtype=torch.uint8, device="cuda")
        out = memory.as_strided(t.shape, (apart, *t.stride()[1:]))
        out.copy_(t)
        return out
    k, v, ks, vs = (far(t, n) for t, n in zip(c.device, (1 << 31, 1 << 31, 1 << 30, (1 << 30) + 1)))
    cache = PagedKVCache(k, v, c.table_dev, ks, vs)
    x = torch.from_numpy(rng.standard_normal((43, (heads + 2 * kv) * dim)).astype(np.float32)).cuda()
    for news in ([1, 1, 1], [33, 1, 9]):
        rows, starts, lens = sum(news), starts_of(news, torch), torch.tensor(contexts, dtype=torch.int32, device="cuda")
        q, out = [torch.empty((rows, heads * dim), device="cuda") for _ in range(2)], [torch.empty((rows, heads * dim), device="cuda") for _ in range(2)]
        for i, into in enumerate((c.cache(), cache)):
            hip.RoPEStorePaged(q[i], x[:rows], into, starts, lens, RotaryPositions(dim))
            hip.PagedAttention(out[i], q[i], into, starts, lens, dim ** -0.5)
        assert torch.equal(*q) and torch.equal(*out)
    for a, b in zip((k, v, ks, vs), c.device):
        assert torch.equal(a, b)


@pytest.mark.parametrize("heads,kv,rows", [(h, kv, n) for h, kv in ((4, 1), (8, 8), (5, 1), (32, 8), (17, 1), (16, 1)) for n in (1, 2, 4, 7, 8)])
def test_sequences_of_up_to_and_over_32_rows(hip, heads, kv, rows):
    """from one row to 136 that share a key head, beside a sequence of one token: every number of passes of 16 rows and both kinds of tiles"""
    import torch
    rng = np.random.default_rng(heads * 10 + rows)
    contexts, news = [333, 90, rows, 1100], [rows, 1, rows, 1]
    c = FourBits(torch, rng, contexts, 16, kv, 64)
    q = torch.from_numpy(rng.standard_normal((sum(news), heads * 64)).astype(np.float32)).cuda()
    lens = torch.tensor(contexts, dtype=torch.int32, device="cuda")
    for window, first in ((0, 0), (100, 3)):
        out = torch.full_like(q, 7.5)
        hip.PagedAttention(out, q, c.cache(), starts_of(news, torch), lens, 0.125, window=window, first=first)
        check(out, c, q, news, contexts, heads, 64, 0.125, window, first)
