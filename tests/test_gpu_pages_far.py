"""GPU: copies of 70000 pages whose offsets pass 2^32 bytes, into four bits, within four bits and back: every page is looked at, in its first block and its last."""
import numpy as np
import pytest

import mx4_oracle as mx

pytestmark = pytest.mark.gpu


def test_every_page_of_a_long_copy(hip):
    import torch
    from tensorsharp_amd import PagedKVCache
    table = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    n, page, dim = 70000, 128, 256
    rng = np.random.default_rng(3)

    def marks(sigma):                                                # [pages, 2, 32]: the first block of a page and its last
        return (sigma * rng.standard_normal((n, 2, 32))).astype(np.float16)
    wide_k, wide_v = (torch.zeros((n, page, 1, dim), dtype=torch.float16, device="cuda") for _ in range(2))               # 4.6 GB each
    host = [marks(1.0), marks(40.0)]
    for t, m in zip((wide_k, wide_v), host):
        m = torch.from_numpy(m).cuda()
        t[:, 0, 0, :32], t[:, page - 1, 0, dim - 32:] = m[:, 0], m[:, 1]
    codes = [torch.full((n, page, 1, dim // 2), 0x35, dtype=torch.uint8, device="cuda") for _ in range(2)]               # 2.3 GB each
    scales = [torch.full((n, page, 1, dim // 32), 100, dtype=torch.uint8, device="cuda") for _ in range(2)]
    four = PagedKVCache(*codes, table, *scales)
    wide = PagedKVCache(wide_k, wide_v, table)
    to = rng.permutation(n)
    moves = lambda a, b: torch.from_numpy(np.stack([a, b], axis=1).astype(np.int32)).cuda()  # noqa: E731
    hip.CopyPages(four, wide, moves(np.arange(n), to))

    def holds(where):
        """page where[i] has what page i had"""
        for c, s, m in zip(codes, scales, host):
            e = mx.scales(m.astype(np.float64))
            want = mx.pack(mx.codes(m.astype(np.float64), e))
            at = torch.from_numpy(np.ascontiguousarray(where)).cuda()
            (c0, s0), (c1, s1), (c2, s2) = ((c[at, p, 0].cpu().numpy(), s[at, p, 0].cpu().numpy()) for p in (0, page // 2, page - 1))
            assert np.array_equal(s0[:, 0], e[:, 0, 0]) and np.array_equal(s2[:, -1], e[:, 1, 0])
            assert np.array_equal(c0[:, :16], want[:, 0]) and np.array_equal(c2[:, -16:], want[:, 1])
            # (beside and between them are zeros, whose power is the least)
            assert not c0[:, 16:].any() and not c1.any() and not c2[:, :-16].any() and (s1 == 1).all()
    holds(to)
    half = n // 2                                                    # within four bits: the upper half becomes the lower one
    low = np.argsort(to)                                             # what page p holds: that of low[p]
    hip.CopyPages(four, four, moves(np.arange(half), np.arange(half, n)[::-1]))
    now = low.copy()
    now[half:] = low[:half][::-1]
    host = [m[now] for m in host]
    holds(np.arange(n))
    wide_k.fill_(7.0)
    wide_v.fill_(7.0)
    hip.CopyPages(wide, four, moves(np.arange(n), np.arange(n)))
    for t, m in zip((wide_k, wide_v), host):
        want = mx.rounded(m.astype(np.float64)).astype(np.float16)
        assert np.array_equal(t[:, 0, 0, :32].cpu().numpy(), want[:, 0]) and np.array_equal(t[:, page - 1, 0, dim - 32:].cpu().numpy(), want[:, 1])
        assert not t[:, page // 2].any() and not t[:, 0, 0, 32:].any()
    del wide, four, wide_k, wide_v, codes, scales
    torch.cuda.empty_cache()
