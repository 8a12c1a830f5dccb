"""GPU: the operators for many sequences together, as a server's step issues them around the quantized products: QKV projection with its norm,
rotation and store into the cache, attention over the cache, output projection and FFN, sampling.

The step is held against the whole-layer decode of the same weights, token by token over one contiguous cache per sequence: the products differ
by the bounds that the layer tests hold them to (3e-3 of the norm for a layer, fp16 operands in batched calls), attention itself by 1e-5."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, DIM, INTER = 512, 8, 2, 64, 1024


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def make_layer(torch, seed):
    from tensorsharp_amd import QuantizedWeight, synth
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    w = lambda n, k, s: QuantizedWeight(synth.random_weight(8, n, k, "cuda", s), 8, k, n)  # noqa: E731
    vec = lambda n: 1.0 + 0.1 * torch.randn(n, generator=g, device="cuda")  # noqa: E731
    q, k = HEADS * DIM, KV * DIM
    return {"attn_norm": vec(HIDDEN), "ffn_norm": vec(HIDDEN), "q_norm": vec(DIM), "k_norm": vec(DIM), "qkv": w(q + 2 * k, HIDDEN, seed + 1),
            "o": w(HIDDEN, q, seed + 2), "gate_up": w(2 * INTER, HIDDEN, seed + 3), "down": w(HIDDEN, INTER, seed + 4)}


def layer_step(hip, torch, hidden, L, cache, starts, lens, rope):
    """one layer for the new tokens of many sequences, in place on hidden [rows, HIDDEN]"""
    rows = hidden.shape[0]
    qkv = torch.empty((rows, (HEADS + 2 * KV) * DIM), device="cuda")
    hip.UseCurrentStream()
    hip.FusedRmsNormMatMulQuant(qkv, hidden, L["attn_norm"], 1e-6, L["qkv"])
    query = qkv[:, :HEADS * DIM]
    hip.RoPEStorePaged(query, qkv, cache, starts, lens, rope, L["q_norm"], L["k_norm"], 1e-6)
    attended = torch.empty((rows, HEADS * DIM), device="cuda")
    hip.PagedAttention(attended, query, cache, starts, lens, DIM ** -0.5)
    hip.FusedOutProjFFN(hidden, attended, L["o"], L["ffn_norm"], 1e-6, L["gate_up"], L["down"], INTER)


def decode_reference(hip, torch, prompts, L, max_seq):
    """token by token through the whole-layer decode: hidden states and caches of each sequence"""
    out, caches = [], []
    for x in prompts:
        kc, vc = (torch.zeros((KV, max_seq, DIM), device="cuda") for _ in range(2))
        h = x.clone()
        for p in range(len(x)):
            hip.TransformerLayerDecode(h[p], L["attn_norm"], L["qkv"], L["q_norm"], L["k_norm"], L["o"], L["ffn_norm"], L["gate_up"], L["down"], kc, vc,
                                       HEADS, KV, DIM, p, 1e-6, 10000.0, 1.0, 2)
        out.append(h)
        caches.append((kc, vc))
    return out, caches


def i32(torch, v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype,bound", [("float32", 3e-3), ("float16", 3e-3), ("bfloat16", 6e-3)])
def test_prompts_in_chunks_and_answers_in_one_batch(hip, dtype, bound):
    """three prompts read in chunks of different lengths while others are already answered; hidden states as of the decode call (a 16-bit cache
    adds the rounding of its keys and values: 2^-9 of each in bf16, half of the layer's bound)"""
    import torch
    from tensorsharp_amd import PagedKVCache, RotaryPositions
    L = make_layer(torch, 40)
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    lengths = [67, 9, 30]
    prompts = [torch.randn((n, HIDDEN), generator=g, device="cuda") for n in lengths]
    ref, caches = decode_reference(hip, torch, prompts, L, 96)
    pages, page = 12, 16
    k = torch.full((pages, page, KV, DIM), float("nan"), device="cuda").to(getattr(torch, dtype))
    v = torch.full_like(k, float("nan"))
    cache = PagedKVCache(k, v, i32(torch, [[3, 7, 0, 9, 11], [2, -1, -1, -1, -1], [5, 8, -1, -1, -1]]))
    rope = RotaryPositions(DIM, mode=2, base=10000.0)
    done = [0, 0, 0]
    for news in ([40, 0, 1], [26, 8, 20], [1, 1, 9]):
        rows = torch.cat([p[d:d + n] for p, d, n in zip(prompts, done, news)])
        done = [d + n for d, n in zip(done, news)]
        starts = i32(torch, [0] + list(np.cumsum(news)))
        layer_step(hip, torch, rows, L, cache, starts, i32(torch, done), rope)
        at = 0
        for s, n in enumerate(news):
            if n:
                assert rel(rows[at:at + n], ref[s][done[s] - n:done[s]]) <= bound, (news, s)
            at += n
    assert done == lengths
    step = {"float32": 1e-4, "float16": 1e-3, "bfloat16": 4e-3}[dtype]                   # the projection's own bound, and the type's step
    for s, n in enumerate(lengths):
        p = torch.arange(n, device="cuda")
        where = (cache.page_table[s].long()[p // page], p % page)
        for mine, theirs in ((k, caches[s][0]), (v, caches[s][1])):
            assert rel(mine[where].float(), theirs[:, :n].transpose(0, 1)) <= 1e-3 + step


def test_a_prompt_goes_on_in_the_whole_layer_decode(hip):
    """the prompt in one chunk into the contiguous fp32 cache that the decode call takes, then tokens through that call - and back"""
    import torch
    from tensorsharp_amd import PagedKVCache, RotaryPositions
    L = make_layer(torch, 50)
    g = torch.Generator(device="cuda")
    g.manual_seed(8)
    x = torch.randn((60, HIDDEN), generator=g, device="cuda")
    (ref,), _ = decode_reference(hip, torch, [x], L, 64)
    kc, vc = (torch.full((KV, 64, DIM), float("nan"), device="cuda") for _ in range(2))
    cache = PagedKVCache(kc.transpose(0, 1)[None], vc.transpose(0, 1)[None], i32(torch, [[0]]))
    rope = RotaryPositions(DIM, mode=2, base=10000.0)
    h = x.clone()
    layer_step(hip, torch, h[:50], L, cache, i32(torch, [0, 50]), i32(torch, [50]), rope)
    for p in range(50, 55):
        hip.TransformerLayerDecode(h[p], L["attn_norm"], L["qkv"], L["q_norm"], L["k_norm"], L["o"], L["ffn_norm"], L["gate_up"], L["down"], kc, vc,
                                   HEADS, KV, DIM, p, 1e-6, 10000.0, 1.0, 2)
    layer_step(hip, torch, h[55:], L, cache, i32(torch, [0, 5]), i32(torch, [60]), rope)
    for a, b in ((0, 50), (50, 55), (55, 60)):
        assert rel(h[a:b], ref[a:b]) <= 3e-3


def build_step(torch, seqs, seed, vocab=5000, page=16, max_pages=40):
    """what a captured decode step works on: fixed buffers, lengths and tables that change between its replays"""
    from tensorsharp_amd import PagedKVCache, RotaryPositions
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    pages = seqs * max_pages
    s = {"qkv": r(seqs, (HEADS + 2 * KV) * DIM), "query": torch.zeros((seqs, HEADS * DIM), device="cuda"), "out": torch.zeros((seqs, HEADS * DIM), device="cuda"),
         "k": r(pages, page, KV, DIM).half(), "v": r(pages, page, KV, DIM).half(), "logits": 3 * r(seqs, vocab), "u": torch.rand(seqs, generator=g, device="cuda"),
         "temperature": torch.full((seqs,), 0.8, device="cuda"), "top_k": i32(torch, [40] * seqs), "top_p": torch.full((seqs,), 0.9, device="cuda"),
         "tokens": i32(torch, [0] * seqs), "probs": torch.zeros(seqs, device="cuda"), "starts": i32(torch, list(range(seqs + 1))), "lens": i32(torch, [1] * seqs),
         "table": torch.arange(pages, dtype=torch.int32, device="cuda").view(seqs, max_pages).clone(), "rope": RotaryPositions(DIM)}
    s["cache"] = PagedKVCache(s["k"], s["v"], s["table"])
    return s


def step(hip, s):
    hip.RoPEStorePaged(s["query"], s["qkv"], s["cache"], s["starts"], s["lens"], s["rope"])
    hip.PagedAttention(s["out"], s["query"], s["cache"], s["starts"], s["lens"], DIM ** -0.5)
    hip.SampleTokens(s["tokens"], s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], None, s["probs"])


def results(s):
    return [s[n].clone() for n in ("query", "out", "k", "v", "tokens", "probs")]


def change(torch, s, turn, seqs):
    """other lengths, pages, inputs and settings for the next step"""
    g = torch.Generator(device="cuda")
    g.manual_seed(100 + turn)
    s["qkv"].normal_(generator=g)
    s["logits"].normal_(0, 3, generator=g)
    s["u"].uniform_(generator=g)
    s["lens"].copy_(torch.randint(1, 600, (seqs,), generator=g, device="cuda").to(torch.int32))
    s["table"].copy_(torch.randperm(s["table"].numel(), generator=g, device="cuda").to(torch.int32).view_as(s["table"]))
    s["top_k"].fill_([40, 0, 1, 3000][turn % 4])
    s["top_p"].fill_([0.9, 0.5, 1.0][turn % 3])
    s["temperature"].fill_([0.8, 0.0][turn % 5 == 4])


def test_a_captured_step_serves_other_lengths_when_it_is_replayed(hip):
    import torch
    seqs = 6
    s, eager = build_step(torch, seqs, 1), build_step(torch, seqs, 1)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(hip, s)                                                  # the stream's scratch is made by its first call
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):                                            # two graphs that share it
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step(hip, s)
            graphs.append(graph)
    for turn in range(10):
        change(torch, s, turn, seqs)
        change(torch, eager, turn, seqs)
        eager["k"].copy_(s["k"])
        eager["v"].copy_(s["v"])
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[turn % 2].replay()
        step(hip, eager)                                              # (on its own stream, beside the replay)
        torch.cuda.synchronize()
        for a, b in zip(results(s), results(eager)):
            assert torch.equal(a, b), turn


def test_streams_and_threads_beside_one_another(hip):
    """steps on four streams, from four threads, give what they give alone"""
    import threading
    import torch
    states = [build_step(torch, 5 + i, 10 + i) for i in range(4)]
    for i, s in enumerate(states):
        change(torch, s, i, 5 + i)
    alone = []
    for s in states:
        step(hip, s)
        torch.cuda.synchronize()
        alone.append(results(s))
    streams = [torch.cuda.Stream() for _ in states]
    torch.cuda.synchronize()

    def work(s, stream):
        with torch.cuda.stream(stream):
            for _ in range(25):
                step(hip, s)
    threads = [threading.Thread(target=work, args=a) for a in zip(states, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for s, want in zip(states, alone):
        for a, b in zip(results(s), want):
            assert torch.equal(a, b)


def test_row_starts_outside_the_rows_are_cut_off(hip):
    """a batch of fewer rows than its row starts speak of (and one whose first begins in front of it): as if these ended with the rows"""
    import torch
    got = []
    for starts in ([0, 1, 3, 6], [-4, 1, 3, 50]):
        s = build_step(torch, 3, 20)
        s["qkv"] = s["qkv"].repeat(2, 1)
        s["qkv"].add_(torch.arange(6, device="cuda")[:, None] / 7)
        s["query"], s["out"] = (torch.zeros((6, HEADS * DIM), device="cuda") for _ in range(2))
        s["starts"], s["lens"] = i32(torch, starts), i32(torch, [40, 17, 200])
        hip.RoPEStorePaged(s["query"], s["qkv"], s["cache"], s["starts"], s["lens"], s["rope"])
        hip.PagedAttention(s["out"], s["query"], s["cache"], s["starts"], s["lens"], DIM ** -0.5)
        got.append([s[n].clone() for n in ("query", "out", "k", "v")])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert bool(got[0][1].abs().sum(1).min() > 0)


def test_the_likeliest_token_of_a_quantized_head(hip):
    """hidden states through a quantized head into the sampler: greedy rows take the largest logit, top-k 1 as well"""
    import torch
    from tensorsharp_amd import QuantizedWeight, synth
    vocab = 3001
    head = QuantizedWeight(synth.random_weight(8, vocab, HIDDEN, "cuda", 5), 8, HIDDEN, vocab)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    logits = hip.LinearForward(torch.randn((7, HIDDEN), generator=g, device="cuda"), head)
    tokens = i32(torch, [-1] * 7)
    u = torch.rand(7, generator=g, device="cuda")
    temperature = torch.tensor([0.0, 1.0, 0.0, 2.0, 0.0, 0.5, 1.0], device="cuda")
    hip.SampleTokens(tokens, logits, u, temperature, top_k=i32(torch, [0, 1, 5, 1, 0, 1, 1]))
    assert torch.equal(tokens.long(), logits.argmax(1))
