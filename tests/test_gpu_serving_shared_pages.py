"""GPU: a server's steps over pages that sequences share - lengths, copies of begun pages, stores, attention, forks, ends, compaction - with two layers'
caches in four bits and one in 16 bits whose tokens see a window and the first positions.

Beside it every sequence has pages of its own in caches that hold the same values, forked by copying whole sequences: where a page lies and who else has it
changes no number, so results are the same bits."""
import numpy as np
import pytest

from test_gpu_four_bits_layouts import laid_out
from test_gpu_attention_four_bits import starts_of

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, PAGE, ROOM, WINDOW, FIRST = 8, 2, 64, 16, 12, 70, 4


class Server:
    """pools of `seqs` sequences; own: the sequences' own pages, in order"""

    def __init__(self, hip, torch, seqs, pages, own=False):
        from tensorsharp_amd import PagedKVCache, PagePool, RotaryPositions
        self.hip, self.torch, self.seqs, self.own = hip, torch, seqs, own
        i32 = dict(dtype=torch.int32, device="cuda")
        self.table = torch.arange(seqs * ROOM, **i32).view(seqs, ROOM).clone() if own else torch.full((seqs, ROOM), -1, **i32)
        self.lens, self.missing, self.moves = torch.zeros(seqs, **i32), torch.zeros(1, **i32), torch.zeros((seqs, 2), **i32)
        self.pool = None if own else PagePool(self.table, torch.zeros(pages, **i32), self.lens, PAGE)
        pages = seqs * ROOM if own else pages
        four = lambda order: [laid_out(torch, (pages, PAGE, KV, n), order)[0] for n in (DIM // 2, DIM // 2, DIM // 32, DIM // 32)]  # noqa: E731
        nan = lambda: torch.full((pages, PAGE, KV, DIM), float("nan"), device="cuda").half()  # noqa: E731
        parts = [four((0, 1, 2, 3)), four((0, 2, 1, 3))]
        self.caches = [PagedKVCache(k, v, self.table, ks, vs) for k, v, ks, vs in parts] + [PagedKVCache(nan(), nan(), self.table)]
        self.rope = RotaryPositions(DIM)

    def copy(self, moves):
        for c in self.caches:
            self.hip.CopyPages(c, c, moves)

    def grow(self, lengths):
        if self.own:
            self.lens.copy_(lengths)
            return
        self.hip.ResizeSequences(self.pool, lengths, self.moves, self.missing)
        self.copy(self.moves)

    def step(self, x, starts, query, out):
        """x, query, out: of each cache; row_starts"""
        for i, c in enumerate(self.caches):
            self.hip.RoPEStorePaged(query[i], x[i], c, starts, self.lens, self.rope)
            self.hip.PagedAttention(out[i], query[i], c, starts, self.lens, DIM ** -0.5, **(dict(window=WINDOW, first=FIRST) if i == 2 else {}))

    def fork(self, children, parents):
        if not self.own:
            moves = self.torch.zeros((len(children), 2), dtype=self.torch.int32, device="cuda")
            self.hip.ForkSequences(self.pool, children, parents, moves, self.missing)
            return self.copy(moves)
        of = list(range(self.seqs))
        for c, p in zip(children.tolist(), parents.tolist()):
            of[c] = p
        of = self.torch.tensor(of, device="cuda")
        for c in self.caches:
            for t in (c.k, c.v, c.k_scales, c.v_scales):
                if t is not None:
                    t.view(self.seqs, ROOM, *t.shape[1:]).copy_(t.reshape(self.seqs, ROOM, *t.shape[1:])[of]) if t.is_contiguous() else \
                        t.copy_(t.clone().reshape(self.seqs, ROOM, *t.shape[1:])[of].reshape(t.shape))
        self.lens.copy_(self.lens[of])

    def compact(self, most):
        if not self.own:
            moves = self.torch.zeros((most, 2), dtype=self.torch.int32, device="cuda")
            self.hip.CompactPages(self.pool, moves)
            self.copy(moves)


def i32(torch, v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def buffers(torch, rows, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = [torch.randn((rows, (HEADS + 2 * KV) * DIM), generator=g, device="cuda") for _ in range(3)]
    return x, [torch.zeros((rows, HEADS * DIM), device="cuda") for _ in range(3)], [torch.zeros((rows, HEADS * DIM), device="cuda") for _ in range(3)]


@pytest.mark.parametrize("pages", [40, 14, 17000])
def test_many_steps(hip, pages):
    """with pages enough, with so few that steps and forks are refused until a sequence ends, and with more than one workgroup looks after"""
    import torch
    seqs = 6
    shared, alone = Server(hip, torch, seqs, pages), Server(hip, torch, seqs, pages, own=True)
    rng = np.random.default_rng(1)
    lens = np.zeros(seqs, dtype=np.int64)
    refused = 0
    for turn in range(40):
        news = [int(rng.integers(1, 50)) if lens[s] == 0 and rng.random() < 0.6 else int(rng.integers(0, 4)) if lens[s] else 0 for s in range(seqs)]
        news = [n if lens[s] + n <= ROOM * PAGE else 0 for s, n in enumerate(news)]
        shared.grow(i32(torch, (lens + news).tolist()))
        if shared.missing.item():                                     # some sequence has to end, and the step is tried again later
            refused += 1
            lens[int(np.argmax(lens))] = 0
            shared.grow(i32(torch, lens.tolist()))
            alone.grow(i32(torch, lens.tolist()))
            continue
        lens += news
        alone.grow(i32(torch, lens.tolist()))
        assert shared.lens.tolist() == lens.tolist()
        rows = sum(news)
        if rows:
            got = []
            for s in (shared, alone):
                x, query, out = buffers(torch, rows, turn)
                s.step(x, starts_of(news, torch), query, out)
                got.append(out)
            for i, (a, b) in enumerate(zip(*got)):
                assert torch.isfinite(a).all() and torch.equal(a, b), (turn, i)
        if turn % 3 == 2:                                             # beams: some go on from others
            children, parents = i32(torch, rng.permutation(seqs)[:4].tolist()), i32(torch, rng.integers(0, seqs, 4).tolist())
            was = shared.lens.tolist()
            shared.fork(children, parents)
            if shared.missing.item():
                assert shared.lens.tolist() == was
                refused += 1
            else:
                alone.fork(children, parents)
                assert shared.lens.tolist() == alone.lens.tolist()
                lens = np.array(shared.lens.tolist())
        if turn % 7 == 6:                                             # one ends, and the pages are moved together
            lens[int(rng.integers(0, seqs))] = 0
            for s in (shared, alone):
                s.grow(i32(torch, lens.tolist()))
            shared.compact(int(rng.integers(1, 40)))
        held = shared.table[shared.table >= 0]
        assert torch.equal(torch.bincount(held.long(), minlength=pages), shared.pool.references.long()), turn
    assert refused > 0 or pages != 14


def test_a_captured_step_and_two_streams(hip):
    """answers of six sequences, each step captured: lengths, the copies that they ask for, stores and attention; two servers side by side on streams of their own"""
    import torch
    seqs, servers = 6, []
    for i in range(2):
        s, alone = Server(hip, torch, seqs, 60), Server(hip, torch, seqs, 60, own=True)
        news = [20 + 5 * i, 1, 16, 33, 4, 47]
        for one in (s, alone):
            one.grow(i32(torch, news))
            x, query, out = buffers(torch, sum(news), i)
            one.step(x, starts_of(news, torch), query, out)
        pairs = i32(torch, [1, 4]), i32(torch, [0, 5])                # two that share whole pages; their begun pages are copied
        for one in (s, alone):
            one.fork(*pairs)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        x, query, out = buffers(torch, seqs, 100 + i)
        starts, goals = i32(torch, list(range(seqs + 1))), s.lens.clone()
        with torch.cuda.stream(side):
            for one in (s, alone):                                    # (the stream's scratch is made; the last tokens get other keys and values in both)
                one.grow(goals)
                one.step(x, starts, query, out)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                goals.add_(1)
                s.grow(goals)
                s.step(x, starts, query, out)
        servers.append((s, alone, side, graph, x, out, starts, goals, query))   # (all that the graph works on)
    for turn in range(20):
        for s, alone, side, graph, x, out, starts, *_ in servers:
            for t in x:
                t.normal_(generator=torch.Generator(device="cuda").manual_seed(turn))
        torch.cuda.synchronize()
        for s, alone, side, graph, *_ in servers:
            with torch.cuda.stream(side):
                graph.replay()
        for s, alone, side, graph, x, out, starts, *_ in servers:
            want = [torch.zeros_like(o) for o in out]
            alone.lens.add_(1)
            alone.step(x, starts, [torch.zeros_like(o) for o in out], want)
            torch.cuda.synchronize()
            assert s.missing.item() == 0 and torch.equal(s.lens, alone.lens)
            for a, b in zip(out, want):
                assert torch.equal(a, b), turn
