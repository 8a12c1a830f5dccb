"""GPU: what the softmax weights of the attention over pages keep of their bits, and sums at the ends of the types' range.

Bounds.  Where one product makes a score it is exact; the exponent's argument rounds twice relative to the score (the scale in powers of two, the
fused product) and once to its own size, the exponential once: 2^-24 (2 |s| + 4) of each weight, twice that of a result (its sum has the same).  Weights
and their sum add the 2^-20 of sum p |v| of test_gpu_paged_attention.py: all of a row's weights keep that, however small they are against its largest.
The weighted values of a long run of keys are summed in 32 bits, 16 keys and one part of the weights (six products of parts in fp32) at a time: each of these
additions rounds by at most 2^-24 of what is summed by then, which is no more than the whole (`additions`).
Over an fp16 cache a weight's last bit is 2^-24, its rounding 2^-25.  The keys of one step (64 at most) have the weights of its largest score to go by, 2^8 or
more, above 2^14 where that stands out of the step's others by 2^20: 64 x 2^-33 of its share of the row, or 64 x 2^-39 (`same_step`).  Keys of other
steps have weights of their own."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def i32(torch, v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def one_sequence(torch, k, v, page):
    """k, v [positions, kv heads, dim] into pages in reverse order"""
    from tensorsharp_amd import PagedKVCache
    n, kv, dim = k.shape
    pages = -(-n // page)
    put = [torch.zeros((pages, page, kv, dim), dtype=k.dtype, device="cuda") for _ in range(2)]
    for to, t in zip(put, (k, v)):
        padded = torch.zeros((pages * page, kv, dim), dtype=k.dtype, device="cuda")
        padded[:n] = t
        to.copy_(padded.view(pages, page, kv, dim).flip(0))
    return PagedKVCache(*put, torch.arange(pages - 1, -1, -1, dtype=torch.int32, device="cuda")[None])


def attend(hip, torch, q, cache, contexts, scale, sinks=None):
    """a sequence over the same pages for every context"""
    from tensorsharp_amd import PagedKVCache
    out = torch.full_like(q, 7.5)
    seqs = len(contexts)
    starts = np.arange(seqs + 1) * (len(q) // seqs)
    if seqs > 1:
        cache = PagedKVCache(cache.k, cache.v, cache.page_table.expand(seqs, -1).contiguous())
    hip.PagedAttention(out, q, cache, i32(torch, starts), i32(torch, contexts), scale, sinks=sinks)
    return out


def additions(dtype, keys, together):
    """roundings of a run of keys: one that all wavefronts take together, or that at least two share out between them"""
    return 2.0 ** -24 * (keys if together else keys / 2) / 16 * {"float16": 2, "bfloat16": 3, "float32": 6}[dtype]


def same_step(dtype, gap, share, v):
    """gap: by how much the largest score surely stands out of others"""
    return (64 * np.where(gap / np.log(2) > 22, 2.0 ** -39, 2.0 ** -33) * share * np.abs(v).max())[:, None] if dtype == "float16" else 0.0


def definition(q, k, v, position, sink=None):
    """one head; q [rows], k [keys]: the one dimension that is not zero; v [keys, dim].  The result, sum p |v| and the largest p"""
    ref, size, share = np.zeros((len(q),) + v.shape[1:]), np.zeros((len(q),) + v.shape[1:]), np.zeros(len(q))
    for r in range(len(q)):
        s = q[r] * k[:position[r] + 1]
        m = s.max() if sink is None else max(s.max(), sink)
        w = np.exp(s - m)
        total = w.sum() + (0.0 if sink is None else np.exp(sink - m))
        ref[r], size[r], share[r] = w @ v[:position[r] + 1] / total, w @ np.abs(v[:position[r] + 1]) / total, w.max() / total
    return ref, size, share


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("gap", [4.0, 8.0, 12.0, 16.0, 20.0, 23.0, 30.0, 40.0])
@pytest.mark.parametrize("rows,seqs,ctx", [(300, 1, 16384), (4, 4, 16384), (1, 1, 40000), (160, 1, 3000), (50, 1, 60)])
@pytest.mark.parametrize("count", [1, 2])
def test_keys_that_take_nearly_all(hip, dtype, gap, rows, seqs, ctx, count):
    """the first key (or one in the middle), and one that is nine behind it, stand `gap` above the others, which are alike or nearly so, and have the value
    0 or 0.05: what is left of the result is the others', to the last bits of each (256 KV heads leave the keys of 300 rows, or 4 sequences, in one piece)"""
    import torch
    rng = np.random.default_rng(int(gap) + rows)
    kv, dim = (256, 16) if ctx == 16384 else (2, 64)
    heads = [0, kv // 2, kv - 1]
    at = [0, 0, ctx // 2 + 7] if rows < ctx // 2 - 8 else [0, 0, 0]
    k = torch.zeros((ctx, kv, dim), device="cuda")
    v = torch.randn((ctx, kv, dim), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * 0.5 + 1.0
    k[:, heads[1]:, 3] = torch.from_numpy(rng.uniform(-0.5, 0.5, ctx).astype(np.float32)).cuda()[:, None]
    for h, a in zip(heads, at):
        k[a:a + 9 * count:9, h, 3] = gap
        v[a:a + 9 * count:9, h] = 0.0 if h != heads[1] else 0.05
    k, v = (t.to(getattr(torch, dtype)) for t in (k, v))
    q = torch.zeros((rows, kv, dim), device="cuda")
    q[:, :, 3] = torch.from_numpy(rng.choice([1.0, 0.75, 0.5], rows).astype(np.float32)).cuda()[:, None] if rows > 1 else 1.0
    contexts = [ctx - 5 * i for i in range(seqs)]
    cache = one_sequence(torch, k, v, 16)
    out = attend(hip, torch, q.view(rows, -1), cache, contexts, 1.0).view(rows, kv, dim).double().cpu().numpy()
    some = np.unique(np.linspace(0, rows - 1, 12).astype(int))
    position = np.concatenate([np.arange(c - rows // seqs, c) for c in contexts])
    for h in heads:
        kh, vh, qh = k[:, h, 3].double().cpu().numpy(), v[:, h].double().cpu().numpy(), q[some, h, 3].double().cpu().numpy()
        ref, size, share = definition(qh, kh, vh, position[some])
        most = (np.abs(qh) * np.abs(kh).max())[:, None]
        d = np.abs(out[some, h] - ref)
        room = (2.0 ** -23 * (2 * most + 4) + 2.0 ** -20 + additions(dtype, ctx, rows // seqs > 32)) * size + same_step(dtype, (gap - 0.5) * qh, share, vh)
        assert np.all(d <= room), (h, float((d / size).max()))


@pytest.mark.parametrize("gap", [16.0, 23.0, 30.0, 36.0])
@pytest.mark.parametrize("rows,seqs,ctx", [(300, 1, 4000), (4, 4, 4000), (100, 1, 700)])
def test_the_steps_behind_a_key_that_takes_all(hip, gap, rows, seqs, ctx):
    """the first key's value and those of its step (64 keys) are 0: all that is left are weights of other steps, which have all their bits (in fp16 as well)"""
    import torch
    kv, dim = 256, 16
    k = torch.zeros((ctx, kv, dim), device="cuda")
    k[0, :, 3] = gap
    v = torch.randn((ctx, kv, dim), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) * 0.5 + 1.0
    v[:64] = 0.0
    k, v = k.half(), v.half()
    q = torch.zeros((rows, kv, dim), device="cuda")
    q[:, :, 3] = 1.0
    contexts = [ctx - 5 * i for i in range(seqs)]
    out = attend(hip, torch, q.view(rows, -1), one_sequence(torch, k, v, 16), contexts, 1.0).view(rows, kv, dim).double().cpu().numpy()
    position = np.concatenate([np.arange(c - rows // seqs, c) for c in contexts])
    for h in (0, 100, 255):
        ref, size, _ = definition(np.ones(rows), k[:, h, 3].double().cpu().numpy(), v[:, h].double().cpu().numpy(), position)
        room = (2.0 ** -23 * (2 * gap + 4) + 2.0 ** -20 + additions("float16", ctx, rows // seqs > 32)) * size
        assert np.all(np.abs(out[:, h] - ref) <= room), (h, float((np.abs(out[:, h] - ref) / size).max()))


@pytest.mark.parametrize("sink", [-200.0, -30.0, 0.0, 30.0, 60.0, 200.0])
@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("rows,ctx", [(1, 300), (100, 300), (1, 9000)])
def test_a_sink_far_above_or_below_the_scores(hip, dtype, sink, rows, ctx):
    import torch
    rng = np.random.default_rng(7)
    k = torch.zeros((ctx, 2, 64), device="cuda")
    k[:, :, 5] = torch.from_numpy(rng.uniform(-2, 2, (ctx, 2)).astype(np.float32)).cuda()
    k[3, 0, 5] = 25.0
    v = torch.from_numpy(rng.standard_normal((ctx, 2, 64)).astype(np.float32)).cuda() + 1.0
    v[3, 0] = 0.0
    k, v = (t.to(getattr(torch, dtype)) for t in (k, v))
    q = torch.zeros((rows, 2, 64), device="cuda")
    q[:, :, 5] = 1.0
    out = attend(hip, torch, q.view(rows, -1), one_sequence(torch, k, v, 16), [ctx], 1.0, torch.full((2,), sink, device="cuda"))
    out = out.view(rows, 2, 64).double().cpu().numpy()
    for h in range(2):
        kh, vh = k[:, h, 5].double().cpu().numpy(), v[:, h].double().cpu().numpy()
        ref, size, share = definition(np.ones(rows), kh, vh, np.arange(ctx - rows, ctx), sink)
        room = (2.0 ** -23 * (2 * max(abs(sink), 25.0) + 4) + 2.0 ** -20) * size + additions(dtype, ctx, rows > 32) * size + 2.0 ** -126
        room += same_step(dtype, np.full(rows, 23.0 if h == 0 else 0.0), share, vh)
        assert np.all(np.abs(out[:, h] - ref) <= room), h


@pytest.mark.parametrize("dtype,large", [("float16", 65504.0), ("bfloat16", 3.2e38), ("float32", 3.2e38), ("float32", 1e37), ("bfloat16", 1e37)])
@pytest.mark.parametrize("rows,ctx,seqs", [(1, 1, 1), (1, 700, 1), (100, 700, 1), (1, 9000, 1), (3, 5000, 1), (60, 4000, 1), (2, 600, 2)])
def test_values_next_to_the_largest(hip, dtype, large, rows, ctx, seqs):
    """what is averaged is finite, so is the average: keys that count alike (their sum is far beyond the type), and one that takes all"""
    import torch
    rng = np.random.default_rng(3)
    k = torch.zeros((ctx, 4, 64), device="cuda")
    k[:, 1, 0] = torch.from_numpy(np.linspace(-3, 3, ctx).astype(np.float32)).cuda()
    k[:, 2, 0] = torch.from_numpy(np.linspace(40, -40, ctx).astype(np.float32)).cuda()
    v = torch.full((ctx, 4, 64), large, device="cuda")
    v[:, 3] *= torch.from_numpy(rng.choice([-1.0, 1.0, 0.5], (ctx, 64)).astype(np.float32)).cuda()
    k, v = (t.to(getattr(torch, dtype)) for t in (k, v))
    q = torch.zeros((rows, 4, 64), device="cuda")
    q[..., 0] = 1.0
    contexts = [ctx - 3 * i for i in range(seqs)]
    out = attend(hip, torch, q.view(rows, -1), one_sequence(torch, k, v, 16), contexts, 1.0).view(rows, 4, 64).double().cpu().numpy()
    position = np.concatenate([np.arange(c - rows // seqs, c) for c in contexts])
    for h in range(4):
        kh, vh = k[:, h, 0].double().cpu().numpy(), v[:, h].double().cpu().numpy()
        ref, size, _ = definition(np.ones(rows), kh, vh, position)
        assert np.all(np.abs(out[:, h] - ref) <= (2.0 ** -23 * (2 * 40 + 4) + 2.0 ** -20 + additions(dtype, ctx, rows // seqs > 32)) * size), h


@pytest.mark.parametrize("dtype,tiny", [("bfloat16", 1e-34), ("bfloat16", 1e-36), ("float32", 1e-30), ("float32", 1e-32)])
@pytest.mark.parametrize("rows,ctx,seqs", [(1, 1, 1), (1, 700, 1), (100, 700, 1), (1, 9000, 1), (60, 4000, 1)])
def test_values_next_to_the_smallest(hip, dtype, tiny, rows, ctx, seqs):
    """weighted by what they have of a row, values and their parts (2^-8 and 2^-16 of them in fp32) stay above the smallest normal number, 1.2e-38"""
    import torch
    rng = np.random.default_rng(4)
    k = torch.zeros((ctx, 2, 64), device="cuda")
    k[:, :, 0] = torch.from_numpy(rng.uniform(-1, 1, (ctx, 2)).astype(np.float32)).cuda()
    v = torch.from_numpy((rng.uniform(0.5, 1.5, (ctx, 2, 64)) * tiny).astype(np.float32)).cuda()
    k, v = (t.to(getattr(torch, dtype)) for t in (k, v))
    q = torch.zeros((rows, 2, 64), device="cuda")
    q[..., 0] = 1.0
    out = attend(hip, torch, q.view(rows, -1), one_sequence(torch, k, v, 16), [ctx], 1.0).view(rows, 2, 64).double().cpu().numpy()
    for h in range(2):
        kh, vh = k[:, h, 0].double().cpu().numpy(), v[:, h].double().cpu().numpy()
        ref, size, _ = definition(np.ones(rows), kh, vh, np.arange(ctx - rows, ctx))
        assert np.all(np.abs(out[:, h] - ref) <= (2.0 ** -23 * (2 + 4) + 2.0 ** -20 + additions(dtype, ctx, rows > 32)) * size), h
