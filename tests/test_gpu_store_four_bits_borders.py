"""GPU: keys that lie closer to a border between two codes, or between two powers, than 32 bits can say go to their own side of it.

A key of pair (b, d) is turned by 2^-20: b (1 - 2^-41) for d = 0, which is below b, and 2^-30 above it for d = -2^-10 (times the block's power); both are b in 32 bits."""
import numpy as np
import pytest

import mx4_oracle as mx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", [0, 2])
@pytest.mark.parametrize("dim", [32, 96, 256])
def test_keys_next_to_borders(hip, dim, mode):
    import torch
    from tensorsharp_amd import PagedKVCache, RotaryPositions
    other = 1 if mode == 0 else 2                                    # what the first dimension is turned with
    rows = []
    for power in (-126, -60, 0, 3, 100):
        for border in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0):
            for sign in (1.0, -1.0):
                for d in (0.0, -2.0 ** -10):
                    x = np.zeros(dim)
                    x[np.arange(4, dim)] = np.tile([0.5, -1.0, 6.0, 3.0], dim // 4 - 1)
                    x[0], x[other] = sign * border, sign * d
                    rows.append(x * 2.0 ** power)
    x = np.stack(rows)
    assert np.array_equal(x.astype(np.float32).astype(np.float64), x)
    want = x.copy()
    c, s = np.cos(2.0 ** -20), np.sin(2.0 ** -20)
    want[:, 0], want[:, other] = x[:, 0] * c - x[:, other] * s, x[:, 0] * s + x[:, other] * c
    assert np.all(want[:, 0] != x[:, 0]) and np.array_equal(want[:, 0].astype(np.float32).astype(np.float64), x[:, 0])
    n = len(x)
    qkv = np.zeros((n, 3 * dim), dtype=np.float32)                   # query, key, value
    qkv[:, dim:2 * dim] = x
    put = lambda *shape: torch.zeros(shape, dtype=torch.uint8, device="cuda")  # noqa: E731
    k, v, ks, vs = put(n, 1, 1, dim // 2), put(n, 1, 1, dim // 2), put(n, 1, 1, dim // 32), put(n, 1, 1, dim // 32)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = PagedKVCache(k, v, torch.arange(n, dtype=torch.int32, device="cuda")[None].contiguous(), ks, vs)
    query = torch.zeros((n, dim), device="cuda")
    rope = RotaryPositions(4, mode=mode, base=2.0 ** 40, freq_scale=2.0 ** -20)          # (the second pair turns by 2^-40: zeros)
    want[:, [i for i in range(4) if i not in (0, other)]] = 0.0
    hip.RoPEStorePaged(query, torch.from_numpy(qkv).cuda(), cache, i32([0, n]), i32([n]), rope, positions=i32([1] * n))
    e = mx.scales(want)
    assert np.array_equal(ks.cpu().numpy()[:, 0, 0], e)
    assert np.array_equal(mx.unpack(k.cpu().numpy()[:, 0, 0]), mx.codes(want, e))
