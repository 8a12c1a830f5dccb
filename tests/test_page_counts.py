"""CPU: sizes and counts of more than 32 bits, of which the calls would take the lower ones, are refused by the facade (on tensors without memory)."""
from types import SimpleNamespace

import pytest
import torch

from tensorsharp_amd import HipBasicOps, PagedKVCache, PagePool
from tensorsharp_amd.hip_basic_ops import _pairs


def meta(*shape, dtype=torch.int32):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("page_size", [2 ** 31, 2 ** 32 + 16, -2 ** 32 + 16, 0, -1])
def test_page_sizes_of_a_pool(page_size):
    with pytest.raises(ValueError, match="page size of 1 to"):
        PagePool(meta(2, 3), meta(8), meta(2), page_size)


@pytest.mark.parametrize("table", [(2, 2 ** 32 + 3), (2 ** 32 + 3, 2), (1, 2 ** 31)])
def test_tables(table):
    with pytest.raises(ValueError, match=r"fewer than 2\^31 sequences and pages"):
        PagePool(meta(*table), meta(8), meta(table[0]), 16)
    k = meta(4, 16, 1, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match=r"fewer than 2\^31 tokens of a page, heads, sequences"):
        PagedKVCache(k, k, meta(*table))


@pytest.mark.parametrize("shape", [(1, 2 ** 32 + 16, 1, 64), (1, 16, 2 ** 31, 64)])
def test_pages(shape):
    k = meta(*shape, dtype=torch.float16)
    with pytest.raises(ValueError, match=r"fewer than 2\^31 tokens of a page, heads"):
        PagedKVCache(k, k, meta(1, 1))


@pytest.mark.parametrize("count", [2 ** 31, 2 ** 32 + 3])
def test_lists(count):
    caches = SimpleNamespace(device=-1)
    with pytest.raises(ValueError, match=r"fewer than 2\^31 pairs"):
        HipBasicOps.CopyPages(caches, caches, meta(count, 2))
    pool = SimpleNamespace(device=-1, _moves=lambda moves, n: _pairs(moves, n, -1))
    with pytest.raises(ValueError, match=r"fewer than 2\^31 pairs"):
        HipBasicOps.CompactPages(pool, meta(count, 2))
    with pytest.raises(ValueError, match=r"fewer than 2\^31 pairs"):
        HipBasicOps.ForkSequences(pool, meta(count), meta(count), meta(count, 2), meta(1))
