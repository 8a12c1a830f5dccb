"""Who has which pages of a cache, kept page by page with plain lists, for the tests."""
import numpy as np


class Pages:
    def __init__(self, table, references, lens, page):
        self.table, self.references, self.lens = np.array(table), np.array(references), np.array(lens)
        self.page = page

    def count(self, tokens):
        return min(self.table.shape[1], -(-max(0, int(tokens)) // self.page))

    def _is(self, e):
        return 0 <= e < len(self.references)

    def _drop(self, e):
        if self._is(e):
            self.references[e] -= 1

    def _free(self, n):
        free = np.flatnonzero(self.references == 0)
        return free[:n].tolist(), max(0, n - len(free))

    def resize(self, lengths):
        """-> moves, missing"""
        most = self.table.shape[1] * self.page
        goals = [int(self.lens[s]) if n < 0 else min(int(n), most) for s, n in enumerate(lengths)]
        for s, goal in enumerate(goals):
            if goal < self.lens[s]:
                for j in range(self.count(goal), self.count(self.lens[s])):
                    self._drop(self.table[s, j])
                    self.table[s, j] = -1
                self.lens[s] = goal
        asks = []
        for s, goal in enumerate(goals):
            if goal > self.lens[s]:
                held = self.count(self.lens[s])
                begun = held > 0 and self.lens[s] % self.page and self._is(self.table[s, held - 1]) and self.references[self.table[s, held - 1]] > 1
                asks += [(s, held - 1, True)] * bool(begun) + [(s, j, False) for j in range(held, self.count(goal))]
        pages, missing = self._free(len(asks))
        if missing:
            return [], missing
        moves = []
        for (s, j, own), page in zip(asks, pages):
            if own:
                moves.append((int(self.table[s, j]), page))
                self._drop(self.table[s, j])
            self.table[s, j] = page
            self.references[page] = 1
        for s, goal in enumerate(goals):
            self.lens[s] = max(goal, self.lens[s])
        return moves, 0

    def fork(self, children, parents):
        seqs = len(self.lens)
        of = list(range(seqs))
        for c, p in zip(children, parents):
            if 0 <= c < seqs and 0 <= p < seqs:
                of[c] = int(p)
        old_table, old_lens = self.table.copy(), self.lens.copy()
        keeps, asks = {}, []
        for s in range(seqs):                                        # (the parent itself first, then the lowest)
            if of[s] == s:
                keeps[s] = s
        for s in range(seqs):
            keeps.setdefault(of[s], s)
        for s in range(seqs):
            p = of[s]
            held = self.count(old_lens[p])
            if keeps[p] != s and held and old_lens[p] % self.page and old_lens[p] <= self.table.shape[1] * self.page and self._is(old_table[p, held - 1]):
                asks.append((s, held - 1))
        pages, missing = self._free(len(asks))
        if missing:
            return [], missing
        moves = []
        for s in range(seqs):
            if of[s] != s:
                for j in range(self.count(old_lens[s])):
                    self._drop(old_table[s, j])
                self.table[s] = -1
                held = self.count(old_lens[of[s]])
                self.table[s, :held] = old_table[of[s], :held]
                self.lens[s] = old_lens[of[s]]
        for (s, j), page in zip(asks, pages):
            moves.append((int(self.table[s, j]), page))
            self.table[s, j] = page
        for s in range(seqs):
            if of[s] != s:
                for j in range(self.count(self.lens[s])):
                    if self._is(self.table[s, j]):
                        self.references[self.table[s, j]] += 1
        return moves, 0

    def compact(self, room):
        used = int((self.references > 0).sum())
        holes = [p for p in range(used) if self.references[p] <= 0]
        tops = [p for p in range(len(self.references) - 1, used - 1, -1) if self.references[p] > 0]
        moves = list(zip(tops, holes))[:room]
        for a, b in moves:
            self.references[b], self.references[a] = self.references[a], 0
        new = dict(moves)
        for s in range(len(self.lens)):
            for j in range(self.count(self.lens[s])):
                self.table[s, j] = new.get(int(self.table[s, j]), self.table[s, j])
        return moves


def random_pages(rng, seqs, max_pages, page, num_pages, share=0.5):
    """A pool that calls may leave: sequences of various lengths, some of which have whole pages, and here and there a begun one, in common"""
    table = np.full((seqs, max_pages), -1, dtype=np.int32)
    lens = np.zeros(seqs, dtype=np.int32)
    free = rng.permutation(num_pages).tolist()
    for s in range(seqs):
        n = int(rng.integers(0, max_pages * page + 1)) if rng.random() < 0.9 else 0
        at = 0
        if s and rng.random() < share:
            p = int(rng.integers(0, s))
            at = min(int(lens[p]) // page if rng.random() < 0.8 else -(-int(lens[p]) // page), -(-n // page))
            table[s, :at] = table[p, :at]
        need = max(0, -(-n // page) - at)
        if need > len(free):
            n, need = min(n, at * page), 0
            table[s, -(-n // page):] = -1
        for j in range(need):
            table[s, at + j] = free.pop()
        lens[s] = n
    references = np.zeros(num_pages, dtype=np.int32)
    for s in range(seqs):
        for j in range(-(-int(lens[s]) // page)):
            references[table[s, j]] += 1
    return Pages(table, references, lens, page)
