"""The life of pages on the GPU against plain lists, and copies of pages between caches."""
import numpy as np
import pytest
import torch

import mx4_oracle as mx
from pages_oracle import Pages, random_pages

pytestmark = pytest.mark.gpu


class Pool:
    """what `pages` says, on the device, with an entry behind each array that no call may change"""

    def __init__(self, hip, pages, apart=0):
        from tensorsharp_amd import PagePool
        seqs, room = pages.table.shape
        self.hip, self.pages = hip, pages
        wide = torch.full((seqs, room + apart), 77, dtype=torch.int32, device="cuda")
        self.table = wide[:, :room]
        self.table.copy_(torch.from_numpy(pages.table.astype(np.int32)))
        self.wide, self.room = wide, room
        self.references = torch.from_numpy(pages.references.astype(np.int32)).cuda()
        self.lens = torch.from_numpy(pages.lens.astype(np.int32)).cuda()
        self.missing = torch.full((1,), -5, dtype=torch.int32, device="cuda")
        self.pool = PagePool(self.table, self.references, self.lens, pages.page)

    def same(self):
        assert torch.equal(self.table.cpu(), torch.from_numpy(self.pages.table.astype(np.int32)))
        assert torch.equal(self.references.cpu(), torch.from_numpy(self.pages.references.astype(np.int32)))
        assert torch.equal(self.lens.cpu(), torch.from_numpy(self.pages.lens.astype(np.int32)))
        assert bool((self.wide[:, self.room:] == 77).all())

    def _listed(self, moves, expected):
        want = np.full(moves.shape, -1, dtype=np.int32)
        want[:len(expected)] = np.array(expected, dtype=np.int32).reshape(-1, 2)
        assert np.array_equal(moves.cpu().numpy(), want)

    def _i32(self, x):
        return torch.from_numpy(np.asarray(x, dtype=np.int32)).cuda()

    def resize(self, lengths):
        moves = torch.zeros((len(lengths), 2), dtype=torch.int32, device="cuda")
        self.hip.ResizeSequences(self.pool, self._i32(lengths), moves, self.missing)
        expected, missing = self.pages.resize(lengths)
        self._listed(moves, expected)
        assert self.missing.item() == missing
        self.same()
        return moves, missing

    def fork(self, children, parents):
        moves = torch.zeros((len(children), 2), dtype=torch.int32, device="cuda")
        self.hip.ForkSequences(self.pool, self._i32(children), self._i32(parents), moves, self.missing)
        expected, missing = self.pages.fork(children, parents)
        self._listed(moves, expected)
        assert self.missing.item() == missing
        self.same()
        return moves, missing

    def compact(self, room):
        moves = torch.zeros((room, 2), dtype=torch.int32, device="cuda")
        self.hip.CompactPages(self.pool, moves)
        self._listed(moves, self.pages.compact(room))
        self.same()
        return moves


# sequences, entries of a table, tokens of a page, pages: one of each; a few; more sequences than a workgroup has threads; more pages than a step of the
# scan; rows of a table longer than a workgroup's part; more sequences than fit a workgroup's memory; pages up to the end of a step; around what one workgroup does alone
SIZES = [(1, 1, 1, 1), (1, 7, 16, 9), (3, 5, 4, 16), (17, 9, 1, 60), (40, 30, 16, 900), (1500, 4, 8, 4001), (70, 300, 2, 17001), (3, 2500, 2, 40000),
         (5000, 3, 4, 9999), (1024, 5, 16, 4096), (30, 2200, 1, 70002), (9, 900, 3, 32768),
         (1024, 32, 4, 16384), (1000, 32, 2, 16385), (100, 327, 3, 16384), (1025, 16, 4, 8000)]


@pytest.mark.parametrize("seqs,room,page,pages", SIZES)
def test_sequences_get_other_lengths(hip, seqs, room, page, pages):
    rng = np.random.default_rng(seqs + room)
    pool = Pool(hip, random_pages(rng, seqs, room, page, pages), apart=3)
    short = 0
    for turn in range(6):
        to = rng.integers(-1, room * page + 2, seqs) if turn % 2 else pool.pages.lens + rng.integers(-2 * page, 3 * page, seqs)
        keep = rng.random(seqs) < 0.3
        to = np.where(keep, -1, to)
        if turn == 3:
            to[:] = 2 ** 31 - 1                                      # (as much as the table has room for)
        if turn == 4:
            to[:] = np.where(rng.random(seqs) < 0.5, 0, -(2 ** 31))
        short += pool.resize(to)[1] > 0
    assert short > 0 or pages > seqs * room or seqs == 1


@pytest.mark.parametrize("seqs,room,page,pages", SIZES)
def test_sequences_go_on_from_others(hip, seqs, room, page, pages):
    rng = np.random.default_rng(7 * seqs + room)
    pool = Pool(hip, random_pages(rng, seqs, room, page, pages), apart=1)
    for turn in range(6):
        if turn == 0:
            children, parents = np.arange(seqs), rng.permutation(seqs)                   # an exchange: nothing is copied
        elif turn == 1:
            children, parents = np.arange(seqs), np.full(seqs, seqs // 2)
        elif turn == 2:
            children, parents = rng.integers(-1, seqs + 1, 2 * seqs), rng.integers(-1, seqs + 1, 2 * seqs)     # twice, and outside
        elif turn == 3:
            children, parents = np.array([seqs - 1]), np.array([seqs - 1])               # itself
        else:
            children, parents = rng.permutation(seqs)[:max(1, seqs // 2)], rng.integers(0, seqs, max(1, seqs // 2))
        moves, _ = pool.fork(children, parents)
        if turn == 0:
            assert bool((moves == -1).all())
        pool.resize(np.where(rng.random(seqs) < 0.5, pool.pages.lens + rng.integers(-page, page + 1, seqs), -1).clip(-1))


@pytest.mark.parametrize("seqs,room,page,pages", SIZES)
@pytest.mark.parametrize("all_at_once", [True, False])
def test_used_pages_move_to_the_front(hip, seqs, room, page, pages, all_at_once):
    rng = np.random.default_rng(11 * seqs + room)
    pool = Pool(hip, random_pages(rng, seqs, room, page, pages))
    for _ in range(3):
        pool.resize(np.where(rng.random(seqs) < 0.5, 0, -1))
        for _ in range(1 if all_at_once else 3):
            pool.compact(pages if all_at_once else max(1, pages // 7))
        if all_at_once:
            used = pool.pages.references > 0
            assert not used[int(used.sum()):].any()
        pool.resize(rng.integers(-1, room * page + 1, seqs))


def test_a_full_and_an_empty_pool(hip):
    pages = Pages(np.full((3, 4), -1), np.zeros(33, dtype=int), [0, 0, 0], 8)
    pool = Pool(hip, pages)
    pool.compact(5)
    pool.fork([0, 1], [2, 2])
    pool.resize([32, 32, 32])
    pages = Pages(np.arange(32).reshape(4, 8), np.ones(32, dtype=int), [64, 64, 64, 63], 8)
    pool = Pool(hip, pages)
    pool.compact(5)
    assert pool.fork([0], [3])[1] == 1                               # a page short: nothing changes
    pool.resize([-1, 8, -1, -1])
    assert pool.fork([0], [3])[1] == 0


def test_two_that_share_a_begun_page_and_go_on_get_one_each(hip):
    pages = Pages([[3, 5, -1], [3, 5, -1], [0, -1, -1]], [1, 0, 0, 2, 0, 2, 0], [12, 12, 3], 8)
    pool = Pool(hip, pages)
    moves, _ = pool.resize([13, 17, -1])
    assert moves.tolist() == [[5, 1], [5, 2], [-1, -1]] and pool.references[5] == 0


def test_entries_that_are_no_pages_are_left_alone(hip):
    pages = Pages([[2, -7, 1, -1], [9, 10 ** 9, -1, -1], [-1, -1, -1, -1]], [0, 1, 1, 0, 0, 0, 0, 0], [10, 7, 0], 4)
    pool = Pool(hip, pages)
    pool.fork([2], [0])
    pool.resize([2, 8, 3])
    pool.compact(3)
    pool.resize([0, 0, 0])


def test_a_captured_step_grows_and_forks_as_lists_say(hip):
    """forks, growth and copies of the begun pages in one graph, replayed over changing lists, with eager work between"""
    rng = np.random.default_rng(3)
    seqs, room, page, num = 12, 8, 4, 120
    pool = Pool(hip, random_pages(rng, seqs, room, page, num))
    from tensorsharp_amd import PagedKVCache
    k, v = (torch.randn((num, page, 2, 32), device="cuda").half() for _ in range(2))
    cache = PagedKVCache(k, v, pool.table)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    children, parents, lengths, forked, grown = i32(seqs), i32(seqs), i32(seqs), i32(seqs, 2), i32(seqs, 2)
    children.fill_(-1)
    lengths.fill_(-1)

    def step():
        hip.ForkSequences(pool.pool, children, parents, forked, pool.missing)
        hip.CopyPages(cache, cache, forked)
        hip.ResizeSequences(pool.pool, lengths, grown, pool.missing)
        hip.CopyPages(cache, cache, grown)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        host = [t.float().cpu() for t in (k, v)]
        for _ in range(8):
            c, p = rng.integers(-1, seqs, seqs), rng.integers(0, seqs, seqs)
            n = np.where(rng.random(seqs) < 0.7, rng.integers(0, room * page, seqs), -1)
            children.copy_(pool._i32(c))
            parents.copy_(pool._i32(p))
            lengths.copy_(pool._i32(n))
            graph.replay()
            moves, _ = pool.pages.fork(c, p)
            more, missing = pool.pages.resize(n)
            for a, b in moves + more:
                for t in host:
                    t[b] = t[a]
            side.synchronize()
            pool.same()
            assert pool.missing.item() == missing
            assert all(torch.equal(t.float().cpu(), h) for t, h in zip((k, v), host))


# ---- copies ----------------------------------------------------------------------------------------

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "mx4": torch.uint8}


class Store:
    """a cache of a type with its values as the host knows them [pages, page, heads, dim] (float64), spread out in memory: heads before tokens, gaps"""

    def __init__(self, rng, kind, pages, page, heads, dim, order, fill=True):
        from tensorsharp_amd import PagedKVCache
        self.kind = kind
        x = [rng.standard_normal((pages, page, heads, dim)).astype(np.float32) * 2.0 ** rng.integers(-3, 4, (pages, page, heads, 1)) for _ in range(2)]
        if not fill:
            x = [np.zeros_like(a) for a in x]
        if kind == "mx4":
            e = [mx.scales(a) for a in x]
            c = [mx.codes(a, s) for a, s in zip(x, e)]
            self.host = [mx.values(a, s) for a, s in zip(c, e)]
            self.tensors = [self._put(mx.pack(a), order) for a in c]
            self.scales = [self._put(s, order, 1) for s in e]
        else:
            self.tensors = [self._put(a, order, dtype=TYPES[kind]) for a in x]
            self.host = [t.double().cpu().numpy() for t in self.tensors]
            self.scales = [None, None]
        self.cache = PagedKVCache(*self.tensors, torch.zeros((1, 1), dtype=torch.int32, device="cuda"), *self.scales)

    @staticmethod
    def _put(a, order, gap=16, dtype=None):
        """on the device with `gap` elements behind each row"""
        t = torch.from_numpy(a)
        t = t.to(dtype) if dtype else t
        shape = a.shape if order == "token" else (a.shape[0], a.shape[2], a.shape[1], a.shape[3])
        wide = torch.zeros((*shape[:3], shape[3] + gap), dtype=t.dtype, device="cuda")
        view = wide[..., :shape[3]]
        view = view if order == "token" else view.transpose(1, 2)
        view.copy_(t.cuda())
        return view

    def values(self):
        if self.kind != "mx4":
            return [t.double().cpu().numpy() for t in self.tensors]
        return [mx.values(mx.unpack(t.cpu().numpy()), e.cpu().numpy()) for t, e in zip(self.tensors, self.scales)]


def held(x, kind):
    """what a cache of that type holds of x"""
    if kind == "mx4":
        return mx.rounded(x)
    return torch.from_numpy(x).float().to(TYPES[kind]).double().numpy()


@pytest.mark.parametrize("dst", ["f32", "f16", "bf16", "mx4"])
@pytest.mark.parametrize("src", ["f32", "f16", "bf16", "mx4"])
@pytest.mark.parametrize("page,heads,dim,orders", [(1, 1, 32, "tt"), (5, 3, 64, "th"), (16, 2, 96, "ht"), (24, 8, 128, "hh"), (7, 1, 256, "tt"), (33, 5, 224, "ht")])
def test_pages_of_one_type_go_into_another(hip, src, dst, page, heads, dim, orders):
    rng = np.random.default_rng(dim + page)
    names = {"t": "token", "h": "head"}
    a, b = Store(rng, src, 11, page, heads, dim, names[orders[0]]), Store(rng, dst, 9, page, heads, dim, names[orders[1]])
    moves = [(3, 8), (10, 0), (3, 1), (-1, 2), (11, 3), (4, 9), (0, -1), (5, 4), (2 ** 31 - 1, 5)]
    hip.CopyPages(b.cache, a.cache, torch.tensor(moves, dtype=torch.int32, device="cuda"))
    for got, was, of in zip(b.values(), b.host, a.host):
        want = was.copy()
        for i, o in moves:
            if 0 <= i < 11 and 0 <= o < 9:
                want[o] = held(of[i], dst) if src != dst else of[i]
        assert np.array_equal(got, want, equal_nan=True)
    for got, was in zip(a.values(), a.host):
        assert np.array_equal(got, was)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16", "mx4"])
@pytest.mark.parametrize("dim", [16, 80, 128])
def test_pages_within_a_cache(hip, kind, dim):
    if kind == "mx4" and dim % 32:
        pytest.skip("four bits come in blocks of 32")
    a = Store(np.random.default_rng(dim), kind, 40, 16, 4, dim, "head")
    if kind == "bf16":
        a.tensors[0].view(torch.int16)[7, 3, 1, 2] = 0x7f81                             # a NaN's bits come along
    moves = [(3, 8), (10, 0), (3, 1), (39, 20), (5, 5), (-1, -1)]
    bits = [t.clone() for t in a.tensors]
    hip.CopyPages(a.cache, a.cache, torch.tensor(moves, dtype=torch.int32, device="cuda"))
    for t, was in zip(a.tensors, bits):
        for i, o in moves[:5]:
            was[o] = was[i]
        view = torch.int32 if kind == "f32" else torch.uint8 if kind == "mx4" else torch.int16
        assert torch.equal(t.view(view), was.view(view))


def test_many_pairs_and_pages_beyond_32_bits(hip):
    """offsets of more than 2^32 bytes, and more pairs than a grid's second dimension has room for"""
    from tensorsharp_amd import PagedKVCache
    table = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    n, page, dim = 70000, 128, 256
    k = torch.zeros((n, page, 1, dim), dtype=torch.float16, device="cuda")               # 4.6 GB
    k[:, 0, 0, 0] = torch.arange(n, device="cuda").remainder(2048).half()
    k[:, page - 1, 0, dim - 1] = torch.arange(n, device="cuda").div(2048, rounding_mode="floor").half()
    v = torch.zeros((n, page, 1, dim // 2), dtype=torch.uint8, device="cuda")
    s = torch.full((n, page, 1, dim // 32), 127, dtype=torch.uint8, device="cuda")
    wide, four = PagedKVCache(k, k, table), PagedKVCache(v, v.clone(), table, s, s.clone())
    moves = torch.stack([torch.randperm(n // 2, device="cuda"), torch.arange(n // 2, n, device="cuda")], dim=1).int()
    hip.CopyPages(four, wide, torch.stack([torch.arange(n - 1, -1, -1, device="cuda")] * 2, dim=1).int())
    assert torch.equal(four.k[:, 0, 0, 0] & 15, v[:, 0, 0, 0] & 15)
    last = mx.rounded(np.concatenate([np.zeros(31), [34.0]]))[-1]
    got = mx.values(mx.unpack(four.k[n - 1, page - 1, 0].cpu().numpy()), four.k_scales[n - 1, page - 1, 0].cpu().numpy())
    assert got[-1] == last
    hip.CopyPages(wide, wide, moves)
    assert torch.equal(k[moves[:, 1].long(), 0, 0, 0], k[moves[:, 0].long(), 0, 0, 0])
    assert torch.equal(k[moves[:, 1].long(), page - 1, 0, dim - 1], k[moves[:, 0].long(), page - 1, 0, dim - 1])


def test_every_value_and_border_in_four_bits(hip):
    """largest magnitudes on, next to and between the borders of every power, the halves between codes, infinities and NaN"""
    from tensorsharp_amd import PagedKVCache
    rows = []
    for e in list(range(-149, -120)) + list(range(-3, 4)) + list(range(118, 128)):
        for top in (1.0, 1.5, 1.75, np.nextafter(np.float32(1.75), np.float32(2)), np.nextafter(np.float32(2), np.float32(1))):
            with np.errstate(over="ignore"):
                x = np.float32(np.float64(top) * 2.0 ** e)
            unit = 2.0 ** (e - 2)
            block = np.float32(np.array([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7], dtype=np.float64) * unit)
            block = np.concatenate([block, -block, np.nextafter(block, np.float32(np.inf))])[:31]
            rows.append(np.concatenate([np.minimum(np.abs(block), np.abs(x)) * np.sign(block), [x if len(rows) % 2 else -x]]).astype(np.float32))
    for odd in (np.inf, -np.inf, np.nan, 2.0 ** 127, -3e38):
        rows.append(np.float32([1.0] * 7 + [odd] + [2.0] * 24))
    rows.append(np.zeros(32, np.float32))
    rows.append(np.full(32, -0.0, np.float32))
    x = np.stack(rows)
    k = torch.from_numpy(x).cuda()[:, None, None, :].contiguous()
    n, table = len(x), torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    four = PagedKVCache(*(torch.zeros((n, 1, 1, 16), dtype=torch.uint8, device="cuda") for _ in range(2)), table,
                        *(torch.zeros((n, 1, 1, 1), dtype=torch.uint8, device="cuda") for _ in range(2)))
    each = torch.arange(n, dtype=torch.int32, device="cuda")[:, None].repeat(1, 2).contiguous()
    hip.CopyPages(four, PagedKVCache(k, k, table), each)
    e = four.k_scales.cpu().numpy()[:, 0, 0]
    assert np.array_equal(e, mx.scales(x.astype(np.float64)))
    fine = e[:, 0] != 255
    assert np.array_equal(mx.unpack(four.k.cpu().numpy()[:, 0, 0])[fine], mx.codes(x.astype(np.float64), np.where(e == 255, 127, e).astype(np.uint8))[fine])
    back = torch.empty_like(k)
    hip.CopyPages(PagedKVCache(back, back.clone(), table), four, each)
    assert np.array_equal(back.cpu().numpy()[:, 0, 0].astype(np.float64), mx.rounded(x.astype(np.float64)), equal_nan=True)
