"""Page tables in numpy where pages have holders of several kinds: serving_ref's steps, with a
grow that tells sequences of the table from what is held elsewhere (madi_kv4_rows.kept)."""
import numpy as np

import serving_ref as S

NONE = S.NONE


class Pages(S.Pages):
    def sequences(self, p, c):
        """Those with page p as number c of their pages."""
        return [j for j in range(len(self.lens)) if self.count(self.length(j)) > c and self.table[j, c] == p]

    def copied(self, fits, before, copy):
        """Which sequences append to a copy of their last page."""
        last = {}
        for i in np.flatnonzero(fits):
            n = self.length(i)
            if copy is not False and n % self.page and self.there(self.table[i, n // self.page]):
                last[i] = int(self.table[i, n // self.page])
        out = set()
        for i, p in last.items():
            grow = [j for j in last if last[j] == p]
            if len(grow) == before[p]:
                if i != max(grow, key=lambda j: (self.length(j) % self.page, j)):
                    out.add(i)
            elif before[p] > 1 and (copy or len(self.sequences(p, self.length(i) // self.page)) > 1):
                out.add(i)
        return out

    def grow(self, add, m, copy=None):
        b, reach = len(self.lens), self.table.shape[1] * self.page
        before, old = self.refs.copy(), [self.length(i) for i in range(b)]
        fits = [0 < add[i] <= reach - old[i] for i in range(b)]
        copies = self.copied(fits, before, copy)
        free = [int(p) for p in np.flatnonzero(before == 0)]
        total, asked, rows_asked, rows = len(free), 0, 0, []
        row_off, out = [0], np.full((b, 3), NONE, np.int32)
        self.left_out = 0
        for i in range(b):
            n, a = old[i], int(add[i]) if fits[i] else 0
            need = self.count(n + a) - self.count(n) + (i in copies)
            grows = a > 0 and (need == 0 or asked + need <= total) and rows_asked + a <= m
            asked, rows_asked = asked + need, rows_asked + a
            self.left_out += bool(add[i]) and not grows
            if grows:
                for c in range(self.count(n), self.count(n + a)):
                    self.table[i, c] = free.pop(0)
                    self.refs[self.table[i, c]] = 1
                if i in copies:
                    source, to = int(self.table[i, n // self.page]), free.pop(0)
                    out[i] = source, to, n % self.page
                    self.table[i, n // self.page] = to
                    self.refs[to] = 1
                    self.refs[source] -= 1
                self.lens[i] = n + a
                rows += [(i, p) for p in range(n, n + a)]
            row_off.append(len(rows))
        seq, pos, slot = np.full(m, NONE, np.int32), np.zeros(m, np.int32), np.full(m, NONE, np.int64)
        for r, (i, p) in enumerate(rows):
            q = int(self.table[i, p // self.page])
            seq[r], pos[r], slot[r] = i, p, q * self.page + p % self.page if self.there(q) else NONE
        return np.array(row_off, np.int32), out, seq, pos, slot


class Contents:
    """What the pages hold: a number for every token that a sequence was given, written where a grow
    says and copied as it says."""

    def __init__(self, n_pages, page, b):
        self.pool, self.page = np.zeros((n_pages, page), np.int64), page
        self.tokens, self.given = [[] for _ in range(b)], 0

    def grow(self, copies, seq, slot):
        for source, to, n in copies:
            if source != NONE:
                self.pool[to, :n] = self.pool[source, :n]
        for i, at in zip(seq, slot):
            if i != NONE:
                self.given += 1
                self.pool.reshape(-1)[at] = self.given
                self.tokens[i].append(self.given)

    def trim(self, to):
        self.tokens = [t[:n] for t, n in zip(self.tokens, to)]

    def fork(self, parent, beams):
        self.tokens = [list(self.tokens[i // beams * beams + parent[i // beams, i % beams]]) for i in range(len(self.tokens))]

    def check(self, table, lens):
        for i, tokens in enumerate(self.tokens):
            at = np.arange(int(lens[i]))
            assert self.pool[table[i, at // self.page], at % self.page].tolist() == tokens, i


def holders_of_many_lengths(rng, b, beams, page, max_pages, m, steps):
    """Steps after which last pages have holders of different lengths: (name, argument) one after the other.  `lens`
    is sent in before each."""
    lens = yield
    for step in range(steps):
        lens = yield "grow", (rng.random(b) < (1, 0.8, 0.5)[step % 3]) * rng.integers(1, 4, b)
        if step % 5 == 4:
            lens = yield "grow", np.where(np.arange(b) == rng.integers(b), rng.integers(0, m // 2 + 1), 1)
        # cut down within the last page, mostly; some are ended
        to = np.maximum(lens - (rng.random(b) < 0.4) * rng.integers(0, page // 2, b), 0)
        lens = yield "trim", np.where(rng.random(b) < 0.05, 0, to)
        if step % 2:
            lens = yield "fork", rng.integers(0, beams, (b // beams, beams))
