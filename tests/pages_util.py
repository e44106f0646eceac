"""A paged cache as plain Python numbers: the rows one after another, as the
documentation of llmk_pages_update states the steps.  Each page's contents are
one number."""
import numpy as np


class Plain:
    def __init__(self, rows, max_pages, page_tokens, num_pages):
        self.R, self.P, self.ps, self.N = rows, max_pages, page_tokens, num_pages
        self.table = np.zeros((rows, max_pages), np.int64)  # entries past a row's pages stay
        self.lengths = np.zeros(rows, np.int64)
        self.refs = np.zeros(num_pages, np.int64)
        self.contents = np.arange(num_pages)

    def pages(self, n):
        return -(-int(n) // self.ps)

    def held(self, r):
        return self.table[r, :self.pages(self.lengths[r])]

    def update(self, new=None, parents=None):
        """Returns (granted, whether a request was invalid, whether pages ran out)."""
        R = self.R
        new = np.full(R, -1) if new is None else np.asarray(new)
        parents = np.full(R, -1) if parents is None else np.asarray(parents)
        granted = np.ones(R, np.int64)
        invalid = full = False
        before, tables = self.lengths.copy(), self.table.copy()
        for r in range(R):
            p = parents[r]
            ok = new[r] <= self.P * self.ps
            if p >= 0:
                ok = ok and p < R and p != r and before[r] == 0 and parents[p] < 0
            if not ok:
                granted[r], invalid = 0, True
            elif p >= 0:
                n = before[p] if new[r] < 0 else min(before[p], new[r])
                k = self.pages(n)
                self.table[r, :k] = tables[p, :k]
                self.refs[tables[p, :k]] += 1
                self.lengths[r] = n
        asked = [r for r in range(R) if granted[r] and new[r] >= 0]
        for r in asked:
            if new[r] < self.lengths[r]:
                for e in self.table[r, self.pages(new[r]):self.pages(self.lengths[r])]:
                    self.refs[e] -= 1
                self.lengths[r] = new[r]
        free = list(np.nonzero(self.refs == 0)[0])
        at_start, taken, stopped = self.refs.copy(), 0, False
        for r in asked:
            cur, want = int(self.lengths[r]), int(new[r])
            if want <= cur:
                continue
            last = self.table[r, cur // self.ps] if cur % self.ps else -1
            shared = last >= 0 and at_start[last] > 1
            copy = shared and self.refs[last] > 1
            need = self.pages(want) - self.pages(cur) + copy
            if taken + need > len(free):
                stopped = True
            if stopped and (need or shared):
                granted[r], full = 0, True
                continue
            got = free[taken:taken + need]
            taken += need
            first = self.pages(cur) - copy
            if copy:
                self.refs[last] -= 1
                self.contents[got[0]] = self.contents[last]
            self.table[r, first:first + need] = got
            self.refs[got] = 1
            self.lengths[r] = want
        return granted, invalid, full

    def compact(self):
        used = self.refs > 0
        M = int(used.sum())
        src = [p for p in range(M, self.N) if used[p]]
        dst = [p for p in range(M) if not used[p]]
        to = np.arange(self.N)
        to[src] = dst
        for r in range(self.R):
            k = self.pages(self.lengths[r])
            self.table[r, :k] = to[self.table[r, :k]]
        for s, d in zip(src, dst):
            self.refs[d], self.refs[s] = self.refs[s], 0
            self.contents[d] = self.contents[s]
        return to

    def check(self):
        """What must hold of any cache."""
        n = np.zeros(self.N, np.int64)
        for r in range(self.R):
            np.add.at(n, self.held(r), 1)
        assert np.array_equal(n, self.refs)
