"""GPU: sequences with room for 2^26 pages each, against plain lists."""
import numpy as np
import pytest

from pages_oracle import Pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("room", [2 ** 26, 2 ** 26 - 16])
def test_the_life_of_pages_in_wide_tables(hip, room):
    import torch
    from tensorsharp_amd import PagePool
    seqs, page, pages = 3, 4, 900
    narrow = Pages(np.full((seqs, 400), -1), np.zeros(pages, dtype=np.int64), np.zeros(seqs, dtype=np.int64), page)
    table = torch.full((seqs, room), -1, dtype=torch.int32, device="cuda")
    references, lens, missing = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (pages, seqs, 1))
    pool = PagePool(table, references, lens, page)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731

    def same(moves, expected):
        want = np.full(moves.shape, -1)
        want[:len(expected)] = np.array(expected).reshape(-1, 2)
        assert np.array_equal(moves.cpu().numpy(), want) and missing.item() == 0
        assert np.array_equal(table[:, :400].cpu().numpy(), narrow.table) and bool((table[:, 400:] == -1).all())
        assert np.array_equal(references.cpu().numpy(), narrow.references) and np.array_equal(lens.cpu().numpy(), narrow.lens)
    moves = torch.zeros((seqs, 2), dtype=torch.int32, device="cuda")
    for lengths in ([1001, 30, 7], [-1, 900, 0], [10, 1300, 90]):
        hip.ResizeSequences(pool, i32(lengths), moves, missing)
        same(moves, narrow.resize(lengths)[0])
        hip.ForkSequences(pool, i32([0, 2, 1]), i32([1, 1, 0]), moves, missing)
        same(moves, narrow.fork([0, 2, 1], [1, 1, 0])[0])
        room_for = torch.zeros((5, 2), dtype=torch.int32, device="cuda")
        hip.CompactPages(pool, room_for)
        same(room_for, narrow.compact(5))
