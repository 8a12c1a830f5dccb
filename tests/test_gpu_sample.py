"""GPU: sampled tokens against their definition in 64 bits.  The tokens have to be the same; a probability rounds once to 32 bits and its weight is a
whole multiple of 2^-43 of the largest: 2^-24 + vocab 2^-43 at most, held to 1e-6."""
import numpy as np
import pytest

import paged_oracle as po

pytestmark = pytest.mark.gpu


def run(hip, logits, u, temperature, top_k=None, top_p=None, min_p=None, strided=False):
    import torch
    rows = len(logits)
    x = torch.from_numpy(np.ascontiguousarray(logits, dtype=np.float32)).cuda()
    if strided:
        wide = torch.full((rows, x.shape[1] + 5), 99.0, device="cuda")
        wide[:, 3:3 + x.shape[1]] = x
        x = wide[:, 3:3 + x.shape[1]]
    put = lambda a, t: None if a is None else torch.from_numpy(np.broadcast_to(np.asarray(a, dtype=t), (rows,)).copy()).cuda()  # noqa: E731
    tokens = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    probs = torch.full((rows,), -7.0, device="cuda")
    hip.SampleTokens(tokens, x, put(u, np.float32), put(temperature, np.float32), put(top_k, np.int32), put(top_p, np.float32), put(min_p, np.float32), probs)
    return tokens.cpu().numpy(), probs.cpu().numpy()


def check(hip, logits, u, temperature, top_k=None, top_p=None, min_p=None, strided=False):
    rows = len(logits)
    got, probs = run(hip, logits, u, temperature, top_k, top_p, min_p, strided)
    row = lambda a, d: np.broadcast_to(np.asarray(d if a is None else a), (rows,))  # noqa: E731
    for r in range(rows):
        token, p = po.sample(logits[r], row(u, 0)[r], row(temperature, 0)[r], row(top_k, 0)[r], row(top_p, 1.0)[r], row(min_p, 0.0)[r])
        assert got[r] == token, (r, got[r], token)
        assert abs(probs[r] - p) <= 1e-6 * p, (r, probs[r], p)


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 1000, 4097, 32064, 50001, 128256])
@pytest.mark.parametrize("top_k,top_p,min_p", [(None, None, None), (40, None, None), (None, 0.9, None), (None, None, 0.02), (50, 0.8, 0.01), (1, 1.0, 0.0),
                                               (0, 0.999999, 0.0)])
def test_sampling(hip, vocab, top_k, top_p, min_p):
    rng = np.random.default_rng(vocab)
    logits = rng.standard_normal((6, vocab)).astype(np.float32) * 2
    for r in range(6):
        logits[r, rng.integers(0, vocab, 20)] += rng.uniform(0, 12, 20).astype(np.float32)
    check(hip, logits, [0.0, 0.37, 0.5, 0.9, 0.999999, rng.random()], [1.0, 0.7, 1.5, 0.3, 2.0, 0.0], top_k, top_p, min_p, strided=vocab % 2 == 1)


def test_equal_logits_are_ranked_by_index(hip):
    rng = np.random.default_rng(1)
    logits = rng.integers(0, 4, (40, 5000)).astype(np.float32)
    logits[0] = 0.0
    logits[1] = -0.0
    logits[2, ::2] = -0.0
    k = rng.integers(1, 4000, 40)
    check(hip, logits, rng.random(40), 1.0, top_k=k)
    check(hip, logits, rng.random(40), 0.5, top_p=rng.random(40))
    check(hip, logits, rng.random(40), 1.0, top_k=k, top_p=rng.random(40), min_p=rng.choice([0.0, 0.2, 0.4], 40))
    check(hip, logits, np.zeros(40), 0.0)
    # all alike: sums are whole numbers and every border is met exactly
    flat = np.zeros((33, 1024), dtype=np.float32)
    check(hip, flat, np.arange(33) / 33, 1.0)
    check(hip, flat, np.arange(33) / 64, 1.0, top_p=np.arange(33) / 32)
    got, _ = run(hip, flat, np.arange(33) / 64, 1.0, top_k=512)
    assert got.tolist() == [8 * i for i in range(33)]


def test_values_that_are_no_numbers(hip):
    logits = np.random.default_rng(2).standard_normal((8, 3001)).astype(np.float32)
    logits[0] = -np.inf
    logits[1] = np.nan
    logits[2, :] = np.nan
    logits[2, 2999] = -3.0
    logits[3, 100:] = -np.inf
    logits[4, [5, 77, 2000]] = np.inf
    logits[5, ::3] = np.nan
    logits[6, :] = -3e38
    logits[6, 11] = 3e38
    logits[7, :] = 1e-42
    for kw in ({}, {"top_k": 2}, {"top_p": 0.7}, {"top_k": 700, "top_p": 0.9, "min_p": 0.1}):
        check(hip, logits, [0.3, 0.3, 0.3, 0.99, 0.5, 0.6, 0.9, 0.25], 1.0, **kw)
        check(hip, logits, [0.3, 0.3, 0.3, 0.99, 0.99, 0.6, 0.9, 0.25], 0.0, **kw)
    assert run(hip, logits, 0.5, 1.0)[0][:3].tolist() == [-1, -1, 2999]


def test_settings_outside_their_ranges(hip):
    logits = np.random.default_rng(3).standard_normal((9, 777)).astype(np.float32)
    check(hip, logits, 0.4, 1.0, top_k=[-1, 0, 777, 778, 2 ** 31 - 1, -2 ** 31, 1, 776, 5])
    check(hip, logits, 0.4, 1.0, top_p=[-1.0, 0.0, 1.0, 1.5, np.inf, 1e-9, 0.9999999, 0.5, -np.inf])
    check(hip, logits, 0.4, 1.0, min_p=[-1.0, 0.0, 1.0, 1.5, np.inf, 1e-9, 0.9999999, 0.5, -np.inf])
    check(hip, logits, 0.4, [1e-30, 1e30, 1e-3, -1.0, 0.0, np.inf, 3e38, 1e-42, 0.01])
    low, _ = run(hip, logits, [-1.0, -0.0, 0.0, -np.inf, 0.0, 0.0, 0.0, 0.0, 0.0], 1.0)
    assert low.tolist() == [0] * 9
    high, _ = run(hip, logits, [1.0, 1.5, np.inf, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0], 1.0)
    assert high.tolist() == [776] * 9
    greedy, _ = run(hip, logits, 0.9, np.nan)
    assert greedy.tolist() == logits.argmax(1).tolist()


def test_draws_follow_the_weights(hip):
    """10000 evenly spread numbers take each token as often as its weight says, one more or less at each border"""
    logits = np.random.default_rng(4).standard_normal(50).astype(np.float32)
    n = 10000
    got, _ = run(hip, np.tile(logits, (n, 1)), (np.arange(n) + 0.5) / n, 0.8)
    w = np.exp(logits.astype(np.float64) / np.float32(0.8))
    assert np.all(np.abs(np.bincount(got, minlength=50) - n * w / w.sum()) <= 1.0 + 1e-6)


def test_the_largest_vocabulary(hip):
    rng = np.random.default_rng(5)
    logits = rng.standard_normal((2, 1 << 20)).astype(np.float32)
    check(hip, logits, [0.2, 0.999], 1.0)
    check(hip, logits, [0.2, 0.999], 1.0, top_k=[300000, 64], top_p=[0.5, 0.9])
    assert run(hip, np.zeros((1, 1 << 20), np.float32), 0.5, 1.0)[0][0] == 1 << 19


def test_rows_alone_and_together_give_the_same(hip):
    rng = np.random.default_rng(6)
    logits = (rng.standard_normal((300, 2000)) * 3).astype(np.float32)
    u, t, k, p, m = rng.random(300), rng.uniform(0, 2, 300), rng.integers(0, 100, 300), rng.uniform(0.3, 1.1, 300), rng.uniform(0, 0.1, 300)
    together = run(hip, logits, u, t, k, p, m)[0]
    for r in (0, 7, 299):
        assert run(hip, logits[r:r + 1], u[r], t[r], k[r], p[r], m[r])[0][0] == together[r]
    check(hip, logits, u, t, k, p, m)
