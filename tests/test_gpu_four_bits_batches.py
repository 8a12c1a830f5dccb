"""GPU: attention over caches in four bits in batches of every kind: hundreds of sequences, more of them than workgroups are for, heads that share one key head by the
hundred, results in the queries' place, columns of a wider tensor, contexts of millions of positions.  Bounds as in test_gpu_attention_four_bits.py."""
import numpy as np
import pytest

import paged_oracle as po
from attention_oracle import FourBits
from test_gpu_attention_four_bits import check, run, starts_of
from test_gpu_store_four_bits import four_bits
from test_gpu_rope import NORM, TURN, lengths

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs,most,kv,news", [(70, 900, 2, "answers"), (130, 400, 2, "mixed"), (700, 90, 1, "answers"), (300, 120, 2, "mixed"), (65, 3000, 1, "answers"),
                                               (90, 700, 1, "few prompts")])
def test_hundreds_of_sequences(hip, seqs, most, kv, news):
    import torch
    rng = np.random.default_rng(seqs)
    contexts = rng.integers(1, most, seqs).tolist()
    contexts[3] = most * 4                                            # one that is much longer than the others
    n = {"answers": [1] * seqs, "mixed": rng.integers(0, 30, seqs).tolist(), "few prompts": [90 if s % 31 == 5 else s % 3 for s in range(seqs)]}[news]
    n = [min(a, b) for a, b in zip(n, contexts)]
    heads, dim = 2 * kv, 64
    c = FourBits(torch, rng, contexts, 16, kv, dim, "head")
    q = torch.from_numpy(rng.standard_normal((sum(n), heads * dim)).astype(np.float32)).cuda()
    for window, first in ((0, 0), (64, 2)):
        check(run(hip, torch, c, q, n, contexts, 0.125, window, first), c, q, n, contexts, heads, dim, 0.125, window, first)


@pytest.mark.parametrize("heads,news,contexts", [(160, [1, 3], [500, 77]), (33, [1, 1, 1], [2000, 40, 900]), (128, [1], [4000]), (129, [2, 1], [1500, 64])])
def test_many_heads_of_one_key_head(hip, heads, news, contexts):
    """from a tile that is all of one token to tokens whose rows are in two tiles"""
    import torch
    rng = np.random.default_rng(heads)
    c = FourBits(torch, rng, contexts, 16, 1, 32)
    q = torch.from_numpy(rng.standard_normal((sum(news), heads * 32)).astype(np.float32)).cuda()
    check(run(hip, torch, c, q, news, contexts, 0.2), c, q, news, contexts, heads, 32, 0.2)


@pytest.mark.parametrize("news,contexts", [([1, 1], [3000, 100]), ([40, 1], [2500, 700]), ([200], [300])])
def test_results_in_the_queries_place_and_in_columns_of_a_wider_tensor(hip, news, contexts):
    import torch
    rng = np.random.default_rng(4)
    heads, kv, dim, rows = 8, 2, 128, sum(news)
    c = FourBits(torch, rng, contexts, 16, kv, dim)
    wide = torch.from_numpy(rng.standard_normal((rows, (heads + 2 * kv) * dim)).astype(np.float32)).cuda()
    q = wide[:, :heads * dim]
    plain = run(hip, torch, c, q.contiguous(), news, contexts, 0.1)
    starts, lens = starts_of(news, torch), torch.tensor(contexts, dtype=torch.int32, device="cuda")
    rest = wide[:, heads * dim:].clone()
    hip.PagedAttention(q, q, c.cache(), starts, lens, 0.1)
    assert torch.equal(q, plain) and torch.equal(wide[:, heads * dim:], rest)


@pytest.mark.parametrize("contexts", [[3000001], [9000001, 5], [70000, 2500000, 1, 900000]])
def test_millions_of_positions(hip, contexts):
    """a step of 128 keys counts 65536 of a sequence at most when work is dealt out: what is behind is the last part's"""
    import torch
    from tensorsharp_amd import PagedKVCache
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    page, dim, heads = 256, 32, 2
    counts = [-(-c // page) for c in contexts]
    pages = sum(counts)
    table = torch.full((len(contexts), max(counts)), -1, dtype=torch.int32, device="cuda")
    order, at = torch.randperm(pages, generator=g, device="cuda").int(), 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n]
        at += n
    code = lambda: torch.randint(0, 256, (pages, page, 1, dim // 2), generator=g, device="cuda", dtype=torch.uint8)  # noqa: E731
    k, v = code(), code()
    ks, vs = (torch.randint(124, 127, (pages, page, 1, 1), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2))
    q = torch.randn((len(contexts), heads * dim), generator=g, device="cuda")
    out = torch.empty_like(q)
    hip.PagedAttention(out, q, PagedKVCache(k, v, table, ks, vs), starts_of([1] * len(contexts), torch), torch.tensor(contexts, dtype=torch.int32, device="cuda"), 0.2)
    half = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device="cuda")
    grid = torch.cat([half, -half])

    def values(codes, scales, s):
        ids = table[s, :counts[s]].long()
        c, e = codes[ids].view(-1, dim // 2)[:contexts[s]].long(), scales[ids].view(-1, 1)[:contexts[s]].double()
        return torch.stack([grid[c & 15], grid[c >> 4]], dim=-1).view(-1, dim) * torch.exp2(e - 127)
    for s, n in enumerate(contexts):
        x = q[s].double().view(heads, dim)
        p = torch.softmax(0.2 * (x @ values(k, ks, s).t().contiguous()), dim=1)
        vals = values(v, vs, s)
        want, size = p @ vals, p @ vals.abs()
        # (scores of up to 0.2 sum |q k|, rounded as above: 2 (dim + 12) 2^-24 of it, 15^-5 of a block's largest; sums of up to n / 64 additions in 32 bits of what has its random signs)
        most = 0.2 * float(x.abs().sum(1).max()) * 6
        bound = (2 * most * (dim + 12) * 2.0 ** -24 + 2 * most * 15.0 ** -5 + 8 * 2.0 ** -24 + np.sqrt(n / 64) * 2.0 ** -24 + 2.0 ** -20) * size
        assert bool(((out[s].double().view(heads, dim) - want).abs() <= bound).all()), s


@pytest.mark.parametrize("which", ["q", "k"])
def test_a_norm_of_queries_or_keys_alone(hip, which):
    import torch
    import mx4_oracle as mx
    from tensorsharp_amd import PagedKVCache, RotaryPositions
    rng = np.random.default_rng(9)
    heads, kv, dim, page, rows = 6, 3, 96, 8, 21
    table = rng.permutation(4).astype(np.int32)[None]
    parts = four_bits(torch, 4, page, kv, dim, "token")
    x = rng.standard_normal((rows, (heads + 2 * kv) * dim)).astype(np.float32)
    w = rng.uniform(0.5, 1.5, dim).astype(np.float32)
    query = torch.empty((rows, heads * dim), device="cuda")
    weight = {"%s_norm" % which: torch.from_numpy(w).cuda()}
    hip.RoPEStorePaged(query, torch.from_numpy(x).cuda(), PagedKVCache(*parts[:2], torch.from_numpy(table).cuda(), *parts[2:]), starts_of([rows], torch),
                       torch.tensor([rows], dtype=torch.int32, device="cuda"), RotaryPositions(dim), eps=1e-5, **weight)
    p, split = np.arange(rows), x.astype(np.float64).reshape(rows, heads + 2 * kv, dim)
    for mine, part in (("q", split[:, :heads]), ("k", split[:, heads:heads + kv])):
        y = po.norm(part, w, 1e-5) if mine == which else part
        ref = po.rope(y, p, dim, 2, base=10000.0)
        if mine == "q":
            room = (TURN + NORM) * lengths(y, dim, 2) + NORM * np.abs(y)
            assert np.all(np.abs(query.cpu().numpy().reshape(rows, heads, dim) - ref) <= room)
        else:
            where = table[0, p // page], p % page
            room = 1.01 * 2.0 ** -24 * lengths(y, dim, 2)
            assert mx.holds(parts[0].cpu().numpy()[where], parts[2].cpu().numpy()[where], ref, room.reshape(rows, kv, -1, 32).max(-1))
