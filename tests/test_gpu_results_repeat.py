"""GPU: a call on the same inputs gives the same bits every time: attention over a cache in four bits, many rows of a sequence and few, at every head dimension, its keys
cut into pieces or not; products of MXFP4 weights with activations as two terms."""
import numpy as np
import pytest

from attention_oracle import FourBits
from test_gpu_attention_four_bits import starts_of

pytestmark = pytest.mark.gpu
REPEATS = 24


@pytest.mark.parametrize("group,news,contexts", [(33, [1, 30, 4] * 6, [600] * 18), (8, [1, 2, 3, 4] * 8, [500] * 32), (4, [200, 1], [900, 2000])])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
def test_attention_over_four_bits(hip, dim, group, news, contexts):
    import torch
    rng = np.random.default_rng(dim + group)
    kv = 2
    c = FourBits(torch, rng, contexts, 3, kv, dim)
    q = torch.from_numpy(rng.standard_normal((sum(news), kv * group * dim)).astype(np.float32)).cuda()
    starts, lens = starts_of(news, torch), torch.tensor(contexts, dtype=torch.int32, device="cuda")
    cache = c.cache()
    results = []
    for _ in range(REPEATS):
        out = torch.empty_like(q)
        hip.PagedAttention(out, q, cache, starts, lens, dim ** -0.5)
        results.append(out)
    assert torch.isfinite(results[0]).all()
    for i, r in enumerate(results):
        assert torch.equal(r, results[0]), (i, int((r != results[0]).sum()))


@pytest.mark.parametrize("M,N,K", [(2300, 1000, 1056), (4096, 512, 2880)])
def test_products_of_mxfp4_weights(hip, oracle, M, N, K):
    import torch
    from oracle.oracle import MXFP4
    from tensorsharp_amd import QuantizedWeight
    rng = np.random.default_rng(M)
    wq = oracle.quantize(MXFP4, (rng.standard_normal(N * K) * 0.02).astype(np.float32))
    x = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).cuda()
    weight = QuantizedWeight(torch.from_numpy(wq).cuda(), MXFP4, K, N)
    results = [hip.LinearForward(x, weight) for _ in range(REPEATS)]
    for i, r in enumerate(results):
        assert torch.equal(r, results[0]), (i, int((r != results[0]).sum()))
