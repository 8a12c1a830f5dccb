"""GPU: attention over pages at the ends of what its arguments may be."""
import numpy as np
import pytest

import paged_oracle as po

pytestmark = pytest.mark.gpu


def i32(torch, v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def attend(hip, torch, c, q, news, contexts, scale, window):
    from tensorsharp_amd import PagedKVCache
    out = torch.full_like(q, 7.5)
    hip.PagedAttention(out, q, PagedKVCache(c.k, c.v, c.table_dev), i32(torch, np.concatenate([[0], np.cumsum(news)])), i32(torch, contexts), scale, window=window)
    return out


@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("heads,news,contexts", [(4, [5], [2]), (4, [8, 3, 2], [3, 3, 9]), (4, [60], [20]), (8, [200, 7], [130, 3]), (4, [3], [6000]), (4, [90], [5000])])
def test_a_window_beyond_every_position_is_none(hip, heads, news, contexts, page):
    """with more new tokens than the context holds as well: those in front of the sequence see nothing, the others what they see without a window"""
    import torch
    rng = np.random.default_rng(sum(news))
    c = po.Cache(torch, rng, contexts, page, 2, 64, torch.float16)
    q = torch.from_numpy(rng.standard_normal((sum(news), heads * 64)).astype(np.float32)).cuda()
    want = attend(hip, torch, c, q, news, contexts, 0.125, 0)
    for window in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 30, max(contexts)):
        assert torch.equal(attend(hip, torch, c, q, news, contexts, 0.125, window), want), window
    at = 0
    for n, ctx in zip(news, contexts):
        hidden = max(0, n - ctx)
        assert torch.all(want[at:at + hidden] == 0) and torch.all(want[at + hidden:at + n].abs().sum(1) > 0)
        at += n


@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("n", [1, 100])
def test_windows_behind_the_page_table(hip, n, page):
    """a context far beyond what the table has room for: a window that ends in front of nothing that is there sees nothing"""
    import torch
    rng = np.random.default_rng(n)
    c = po.Cache(torch, rng, [160], page, 2, 64, torch.float16)
    q = torch.from_numpy(rng.standard_normal((n, 256)).astype(np.float32)).cuda()
    for context in (2 ** 31 - 1, 2 ** 31 - 50, 2 ** 30 + 5, 400):
        for window in (1, 64):
            assert torch.all(attend(hip, torch, c, q, [n], [context], 0.125, window) == 0), (context, window)
    # all of them, and the last ones that are there
    everything = attend(hip, torch, c, q, [n], [2 ** 31 - 1], 0.125, 0)
    k, v = c.rows(0)
    ref, _ = po.attend(q.cpu().numpy().astype(np.float64).reshape(n, 4, 64), k, v, np.full(n, 10 ** 6), 0.125)
    assert np.abs(everything.cpu().numpy().reshape(n, 4, 64) - ref).max() < 1e-5
    some = attend(hip, torch, c, q, [n], [200], 0.125, 120)
    ref, _ = po.attend(q.cpu().numpy().astype(np.float64).reshape(n, 4, 64), k, v, np.arange(200 - n, 200), 0.125, 120)
    assert np.abs(some.cpu().numpy().reshape(n, 4, 64) - ref).max() < 1e-5


def test_factors_of_a_rotation_on_another_device_are_refused(hip):
    """(a device number as a second one would give it: one is enough for this test)"""
    import torch
    from tensorsharp_amd import PagedKVCache, RotaryPositions
    rope = RotaryPositions(64, freq_factors=torch.ones(32, device="cuda"))
    x, pages = torch.ones((3, 2, 64), device="cuda"), torch.zeros((2, 4, 1, 64), device="cuda")
    cache = PagedKVCache(pages, pages.clone(), i32(torch, [[0, 1]]))
    query, qkv = torch.zeros((3, 128), device="cuda"), torch.ones((3, 256), device="cuda")
    hip.RoPE(torch.empty_like(x), x, i32(torch, [0, 1, 2]), rope)
    hip.RoPEStorePaged(query, qkv, cache, i32(torch, [0, 3]), i32(torch, [3]), rope)
    rope.device += 1
    with pytest.raises(ValueError, match="freq_factors is not on the device"):
        hip.RoPE(torch.empty_like(x), x, i32(torch, [0, 1, 2]), rope)
    with pytest.raises(ValueError, match="freq_factors is not on the device"):
        hip.RoPEStorePaged(query, qkv, cache, i32(torch, [0, 3]), i32(torch, [3]), rope)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("n,ctx", [(1, 1), (1, 70), (1, 5000), (40, 50), (3, 9)])
def test_scores_of_minus_infinity_alone_give_zero(hip, dtype, n, ctx):
    """one head's keys are all -infinity in a dimension in which the queries are positive, another's are ordinary"""
    import torch
    rng = np.random.default_rng(ctx)
    c = po.Cache(torch, rng, [ctx], 16, 2, 64, getattr(torch, dtype))
    c.k[:, :, 0, 5] = -np.inf
    q = torch.from_numpy(rng.standard_normal((n, 4, 64)).astype(np.float32)).cuda()
    q[:, :, 5] = torch.tensor([1.0, 1.2345, 0.1, 3.0], device="cuda")
    out = attend(hip, torch, c, q.view(n, -1), [n], [ctx], 0.125, 0).cpu().numpy().reshape(n, 4, 64)
    assert np.all(out[:, :2] == 0.0)
    k, v = c.rows(0)
    ref, _ = po.attend(q.cpu().numpy().astype(np.float64)[:, 2:], k[:, 1:], v[:, 1:], np.arange(ctx - n, ctx), 0.125)
    assert np.abs(out[:, 2:] - ref).max() < 1e-5


@pytest.mark.parametrize("n,ctx", [(1, 300), (100, 300), (1, 9000), (5, 6000)])
def test_sinks_of_infinity(hip, n, ctx):
    """-infinity: as without; infinity: it takes all"""
    import torch
    from tensorsharp_amd import PagedKVCache
    rng = np.random.default_rng(n)
    c = po.Cache(torch, rng, [ctx], 16, 2, 64, torch.float16)
    q = torch.from_numpy(rng.standard_normal((n, 256)).astype(np.float32)).cuda()
    want = attend(hip, torch, c, q, [n], [ctx], 0.125, 0)
    out = torch.full_like(q, 7.5)
    sinks = torch.tensor([-np.inf, np.inf, -np.inf, np.inf], dtype=torch.float32, device="cuda")
    hip.PagedAttention(out, q, PagedKVCache(c.k, c.v, c.table_dev), i32(torch, [0, n]), i32(torch, [ctx]), 0.125, sinks=sinks)
    out, want = out.view(n, 4, 64), want.view(n, 4, 64)
    assert torch.equal(out[:, 0::2], want[:, 0::2]) and torch.all(out[:, 1::2] == 0)
