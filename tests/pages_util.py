"""The pages of a cache as the interface defines them, in plain Python, sequence by sequence."""
import numpy as np


class Refused(Exception):
    pass


class Pool:
    def __init__(self, n_pages, page_rows, n_seqs, max_pages):
        self.n_pages, self.P, self.n_seqs, self.ld = n_pages, page_rows, n_seqs, max_pages
        self.refs = np.zeros(n_pages, np.int64)
        self.tables = np.full((n_seqs, max_pages), -1, np.int64)
        self.lens = np.zeros(n_seqs, np.int64)

    def held(self, n):
        return -(-n // self.P)

    def _list(self, seqs):
        if len(set(seqs)) < len(seqs) or any(not 0 <= s < self.n_seqs for s in seqs):
            raise Refused("list")

    def extend(self, seqs, counts=None):
        """Returns the copies (from, to, rows)."""
        counts = [1] * len(seqs) if counts is None else list(counts)
        self._list(seqs)
        if any(c < 0 for c in counts):
            raise Refused("list")
        refs, tables, lens = self.refs.copy(), self.tables.copy(), self.lens.copy()
        free, copies = [p for p in range(self.n_pages) if refs[p] == 0], []
        for s, c in zip(seqs, counts):
            n = int(lens[s])
            new = [None] * (self.held(n + c) - self.held(n))
            last = n // self.P
            copy = n % self.P and c and refs[tables[s, last]] > 1
            if self.held(n + c) > self.ld or len(free) < len(new) + bool(copy):
                raise Refused("pages")
            if copy:
                page = free.pop(0)
                copies.append((int(tables[s, last]), page, n % self.P))
                refs[tables[s, last]] -= 1
                tables[s, last], refs[page] = page, 1
            for i in range(len(new)):
                tables[s, self.held(n) + i] = free.pop(0)
                refs[tables[s, self.held(n) + i]] = 1
            lens[s] = n + c
        self.refs, self.tables, self.lens = refs, tables, lens
        return copies

    def fork(self, src, dst, keep=None):
        self._list(dst)
        if any(not 0 <= s < self.n_seqs or s in dst for s in src) or any(self.lens[d] for d in dst) or any(k < 0 for k in keep or ()):
            raise Refused("list")
        for i, (s, d) in enumerate(zip(src, dst)):
            n = int(self.lens[s] if keep is None else min(keep[i], self.lens[s]))
            for j in range(self.held(n)):
                self.tables[d, j] = self.tables[s, j]
                self.refs[self.tables[s, j]] += 1
            self.lens[d] = n

    def free(self, seqs):
        self._list(seqs)
        for s in seqs:
            for j in range(self.held(int(self.lens[s]))):
                self.refs[self.tables[s, j]] -= 1
                self.tables[s, j] = -1
            self.lens[s] = 0

    def compact(self):
        used = int((self.refs > 0).sum())
        to = dict(zip([p for p in range(used, self.n_pages) if self.refs[p]], [p for p in range(used) if not self.refs[p]]))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.tables = np.array([[to.get(int(p), int(p)) for p in row] for row in self.tables]).reshape(self.tables.shape)
        return [(a, b, self.P) for a, b in to.items()], used

    def sound(self):
        """Every page has as many holders as its count says, and nothing stands behind a sequence's pages."""
        n = np.zeros(self.n_pages, np.int64)
        for s in range(self.n_seqs):
            h = self.held(int(self.lens[s]))
            for j in range(h):
                n[self.tables[s, j]] += 1
            assert (self.tables[s, h:] == -1).all()
        assert np.array_equal(n, self.refs)
