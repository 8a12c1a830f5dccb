"""GPU: attention whose tokens see a window and the first positions of their sequence, over caches of 16 and 32 bits, against its definition in 64 bits.
Bounds as test_gpu_paged_attention.py derives them."""
import numpy as np
import pytest

import paged_oracle as po
from attention_oracle import attend
from test_gpu_attention_four_bits import check, starts_of

pytestmark = pytest.mark.gpu


def run(hip, torch, c, q, news, contexts, scale, window, first, sinks=None, table=None):
    from tensorsharp_amd import PagedKVCache
    out = torch.full((len(q), q.shape[1]), 7.5, device="cuda")
    hip.PagedAttention(out, q, PagedKVCache(c.k, c.v, c.table_dev if table is None else table), starts_of(news, torch),
                       torch.tensor(contexts, dtype=torch.int32, device="cuda"), scale, window=window, sinks=sinks, first=first)
    return out


CASES = [
    # heads, kv heads, dim, type, page, order, contexts, new tokens, sinks
    (32, 8, 128, "float16", 16, "token", [777, 1, 64, 33, 1500], [1, 1, 1, 1, 1], False),
    (32, 8, 128, "float16", 64, "head", [300, 900], [300, 200], True),
    (8, 1, 128, "bfloat16", 24, "token", [200, 513, 40], [150, 1, 40], True),
    (64, 8, 64, "bfloat16", 16, "head", [700, 260, 5], [65, 1, 5], True),
    (6, 2, 64, "float16", 5, "token", [97, 31, 2], [33, 31, 1], False),
    (7, 1, 80, "float16", 100, "head", [250, 90], [9, 33], True),
    (5, 1, 96, "bfloat16", 1, "token", [129, 300], [128, 3], False),
    (4, 4, 112, "float32", 7, "token", [90, 400], [21, 40], False),
    (16, 2, 128, "float32", 4096, "head", [333], [100], False),
    (3, 3, 192, "float16", 16, "token", [70, 300], [70, 1], True),
    (8, 2, 256, "bfloat16", 33, "token", [150, 460], [40, 1], False),
    (4, 2, 256, "float32", 16, "token", [100, 260], [33, 2], True),
    (8, 2, 256, "float16", 16, "head", [150, 460], [65, 1], False),
    (2, 1, 16, "float16", 3, "token", [50, 10], [17, 10], False),
    (6, 2, 192, "float32", 16, "head", [140, 290], [50, 1], False),
    (6, 2, 96, "float32", 16, "head", [140, 290], [50, 1], False),
    (6, 2, 64, "float32", 16, "head", [140, 290], [50, 1], False),
    (6, 2, 192, "bfloat16", 16, "head", [140, 290], [50, 1], False),
    (6, 2, 128, "bfloat16", 16, "head", [340, 290], [50, 1], False),
    (6, 2, 96, "float16", 16, "head", [340, 290], [50, 1], False),
]


@pytest.mark.parametrize("window,first", [(1, 1), (17, 4), (100, 64), (128, 65), (30, 200), (2 ** 31 - 1, 5), (5, 2 ** 31 - 1), (60, 0)])
@pytest.mark.parametrize("heads,kv,dim,dtype,page,order,contexts,news,sunk", CASES)
def test_windows_with_first_positions(hip, heads, kv, dim, dtype, page, order, contexts, news, sunk, window, first):
    import torch
    rng = np.random.default_rng(heads * dim + page)
    c = po.Cache(torch, rng, contexts, page, kv, dim, getattr(torch, dtype), order)
    rows = sum(news)
    q = torch.from_numpy((2.0 * rng.standard_normal((rows + 2, heads * dim))).astype(np.float32)).cuda()
    sinks = torch.from_numpy(rng.standard_normal(heads).astype(np.float32)).cuda() if sunk else None
    out = run(hip, torch, c, q, news, contexts, 1.0 / np.sqrt(dim), window, first, sinks)
    assert torch.all(out[rows:] == 7.5)
    check(out[:rows], c, q[:rows], news, contexts, heads, dim, 1.0 / np.sqrt(dim), window, first, sinks, terms=False)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("news,contexts", [([1], [7000]), ([1, 2, 1], [2500, 90, 4001]), ([40], [2600]), ([300, 1], [2800, 1900])])
def test_keys_cut_into_pieces(hip, dtype, news, contexts):
    import torch
    rng = np.random.default_rng(len(news))
    heads, kv, dim = 8, 2, 128
    c = po.Cache(torch, rng, contexts, 16, kv, dim, getattr(torch, dtype))
    q = torch.from_numpy((2.0 * rng.standard_normal((sum(news), heads * dim))).astype(np.float32)).cuda()
    for window, first in ((1500, 4), (1500, 130), (700, 1000), (3, 2000)):
        out = run(hip, torch, c, q, news, contexts, 1.0 / np.sqrt(dim), window, first)
        check(out, c, q, news, contexts, heads, dim, 1.0 / np.sqrt(dim), window, first, terms=False)


def test_no_window_and_no_first_positions_are_as_before(hip):
    import torch
    rng = np.random.default_rng(4)
    c = po.Cache(torch, rng, [300, 90], 16, 2, 64, torch.float16)
    q = torch.from_numpy(rng.standard_normal((51, 4 * 64)).astype(np.float32)).cuda()
    a = run(hip, torch, c, q, [1, 50], [300, 90], 0.1, 0, 7)
    b = run(hip, torch, c, q, [1, 50], [300, 90], 0.1, 0, 0)
    assert torch.equal(a, b)
    for first in (-1, 2 ** 31):
        with pytest.raises(ValueError):
            run(hip, torch, c, q, [1, 50], [300, 90], 0.1, 5, first)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("news", [[1], [50]])
def test_infinities_and_nan_between_the_first_and_the_window(hip, dtype, news):
    """what lies between them is not seen; what the first positions hold is"""
    import torch
    rng = np.random.default_rng(6)
    n, heads, kv, dim = 500, 4, 2, 128
    c = po.Cache(torch, rng, [n], 16, kv, dim, getattr(torch, dtype))
    q = torch.from_numpy(rng.standard_normal((news[0], heads * dim)).astype(np.float32)).cuda()
    p = np.arange(10, 380)
    at = (torch.from_numpy(c.table[0, p // 16].astype(np.int64)).cuda(), torch.from_numpy(p % 16).cuda())
    c.v[at] = float("nan")
    c.k[at] = float("inf")
    out = run(hip, torch, c, q, news, [n], 0.1, 60, 10)
    k, v = (np.nan_to_num(t, nan=0.0, posinf=0.0) for t in c.rows(0))
    ref, size = attend(q.cpu().numpy().reshape(-1, heads, dim), k, v, np.arange(n - news[0], n), 0.1, 60, 10)
    assert np.all(np.abs(out.cpu().numpy().reshape(-1, heads, dim) - ref) <= 1e-5 * size)
    c.v[int(c.table[0, 0]), 3, 1, 5] = float("inf")
    out = run(hip, torch, c, q, news, [n], 0.1, 60, 10).cpu().numpy().reshape(-1, heads, dim)
    assert np.all(out[:, 2:, 5] == np.inf)
    out[:, 2:, 5] = ref[:, 2:, 5]
    assert np.all(np.abs(out - ref) <= 1e-5 * size)


@pytest.mark.parametrize("page", [1, 3, 5, 7, 11])
@pytest.mark.parametrize("kind", ["float16", "bfloat16", "float32", "four bits"])
def test_pages_where_the_first_positions_end(hip, kind, page):
    """what follows the first positions lies before the end of their last step, on a page before the last one that was looked up"""
    import torch
    from attention_oracle import FourBits
    from test_gpu_attention_four_bits import run as run_four_bits
    rng = np.random.default_rng(page)
    heads, kv, dim = 8, 1, 64
    news, contexts = [40, 70], [1990, 2600]
    four = kind == "four bits"
    c = FourBits(torch, rng, contexts, page, kv, dim) if four else po.Cache(torch, rng, contexts, page, kv, dim, getattr(torch, kind))
    q = torch.from_numpy((2.0 * rng.standard_normal((sum(news), heads * dim))).astype(np.float32)).cuda()
    for first in (1729, 1793, 1857, 1921, 1900, 900):
        for window in (90, 700):
            out = (run_four_bits if four else run)(hip, torch, c, q, news, contexts, 0.125, window, first)
            check(out, c, q, news, contexts, heads, dim, 0.125, window, first, terms=four)
