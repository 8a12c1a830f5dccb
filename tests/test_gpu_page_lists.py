"""GPU: lists of moves and of forks with as many pairs as a call takes, 2^31 - 1: all of them are read and written, and nothing behind them."""
import numpy as np
import pytest

from pages_oracle import Pages

pytestmark = pytest.mark.gpu
MOST = 2 ** 31 - 1
BEHIND = 4096                                                        # pairs behind a list that stay as they are


def pool_of(torch, pages):
    from tensorsharp_amd import PagePool
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()  # noqa: E731
    table, references, lens = put(pages.table), put(pages.references), put(pages.lens)
    return PagePool(table, references, lens, pages.page), lambda: all(
        np.array_equal(t.cpu().numpy(), want) for t, want in ((table, pages.table), (references, pages.references), (lens, pages.lens)))


def held_by(seqs, room, pages, lens, page):
    """sequences with pages of their own, the last ones first"""
    table, references = np.full((seqs, room), -1, dtype=np.int32), np.zeros(pages, dtype=np.int32)
    at = pages
    for s, n in enumerate(lens):
        for j in range(-(-n // page)):
            at -= 1
            table[s, j], references[at] = at, 1
    return Pages(table, references, lens, page)


def listed(torch, moves, expected):
    got = moves[:len(expected)].cpu().numpy().tolist()
    assert got == [list(m) for m in expected]
    for i in range(len(expected), len(moves), 1 << 28):              # (a comparison of all at once would take as much memory again)
        assert bool((moves[i:i + (1 << 28)] == -1).all()), i


@pytest.mark.parametrize("seqs,pages", [(3, 40), (3, 20000)])
def test_a_compaction_with_room_for_every_move(hip, seqs, pages):
    import torch
    expected = held_by(seqs, 8, pages, [100, 33, 16], 16)
    whole = torch.full((MOST + BEHIND, 2), 7, dtype=torch.int32, device="cuda")          # 16 GiB
    pool, same = pool_of(torch, expected)
    hip.CompactPages(pool, whole[:MOST])
    moves = expected.compact(MOST)
    listed(torch, whole[:MOST], moves)
    assert same() and bool((whole[MOST:] == 7).all())
    del whole
    torch.cuda.empty_cache()


@pytest.mark.parametrize("seqs", [3, 4200])
def test_a_fork_of_every_pair(hip, seqs):
    """most pairs name no sequence; the last ones do"""
    import torch
    lens = [100, 33, 20] + [0] * (seqs - 3)
    expected = held_by(seqs, 8, 60, lens, 16)
    whole = torch.full((MOST + BEHIND, 2), 7, dtype=torch.int32, device="cuda")
    children, parents = (torch.full((MOST,), -1, dtype=torch.int32, device="cuda") for _ in range(2))          # 8 GiB each
    pairs = [(0, 1, 2), (5, 2, 1), (MOST - 2, 1, 0), (MOST - 1, seqs, 0)]
    for i, c, p in pairs:
        children[i], parents[i] = c, p
    missing = torch.full((1,), -5, dtype=torch.int32, device="cuda")
    pool, same = pool_of(torch, expected)
    hip.ForkSequences(pool, children, parents, whole[:MOST], missing)
    moves, short = expected.fork([c for _, c, _ in pairs], [p for _, _, p in pairs])
    listed(torch, whole[:MOST], moves)
    assert missing.item() == short == 0 and same() and bool((whole[MOST:] == 7).all())
    del whole, children, parents
    torch.cuda.empty_cache()
