"""A pool of pages and its operations, one entry at a time on the host."""
import numpy as np


class Pool:
    def __init__(self, n_pages, page, n_seq, stride):
        self.n_pages, self.page, self.n_seq, self.stride = n_pages, page, n_seq, stride
        self.refs = np.zeros(n_pages, np.int32)
        self.table = np.full((n_seq, stride), -1, np.int32)
        self.kv_len = np.zeros(n_seq, np.int32)

    def _pages(self, tokens):
        return -(-int(tokens) // self.page)

    def _length(self, s):
        return min(max(int(self.kv_len[s]), 0), self.stride * self.page)

    def _entries(self, s, n):
        return [int(i) if 0 <= i < self.n_pages else -1 for i in self.table[s, :n]]

    def fork(self, parent=None, keep=None, grow=0, window=0, sinks=0):
        """(copies, result); grow: a number or one for each sequence."""
        n, page, cap = self.n_seq, self.page, self.stride * self.page
        old = [self._entries(s, self._pages(self._length(s))) for s in range(n)]
        rows, keeps, sizes = [], [], []
        for s in range(n):
            p = s if parent is None else int(parent[s])
            p = p if 0 <= p < n else -1
            has = self._length(p) if p >= 0 else 0
            k = has if keep is None else min(max(int(keep[s]), 0), has)
            g = int(grow if np.isscalar(grow) else grow[s])
            row = self._entries(p, self._pages(k)) if p >= 0 else []
            for j in range(len(row)):  # a page all of whose tokens lie behind the window, and are no sinks
                if window and (j + 1) * page - 1 <= k - window and j * page >= sinks:
                    row[j] = -1
            rows.append(row)
            keeps.append(k)
            sizes.append(k + min(max(g, 0), cap - k))
        refs = self.refs.copy()
        for group, by in ((old, -1), (rows, 1)):
            for row in group:
                for i in row:
                    if i >= 0:
                        refs[i] += by
        writers = {}
        for s in range(n):
            if keeps[s] % page and sizes[s] > keeps[s] and rows[s][-1] >= 0:
                writers.setdefault(rows[s][-1], []).append(s)
        copied = {s: i for i, w in writers.items() for s in (w if refs[i] > len(w) else w[1:])}
        for s, i in copied.items():
            rows[s].pop()
        after = refs.copy()
        for i in copied.values():
            after[i] -= 1
        free = [i for i in range(self.n_pages) if refs[i] == 0]
        need = sum(self._pages(z) - len(r) for z, r in zip(sizes, rows))
        if need > len(free):
            return [], (len(free) - need, 0)
        left = len(free) - need
        copies = []
        for s in range(n):
            while len(rows[s]) < self._pages(sizes[s]):
                i = free.pop(0)
                after[i] = 1
                if s in copied and len(rows[s]) == keeps[s] // page:
                    copies.append((copied[s], i, keeps[s] % page))
                rows[s].append(i)
        for s in range(n):
            p = s if parent is None else int(parent[s])
            m = max(len(rows[s]), len(old[s]))
            row = rows[s] + [-1] * (m - len(rows[s]))
            if p == s:  # its kept entries stay as they are, ids of no page among them
                row = [int(self.table[s, j]) if x == -1 and j < self._pages(keeps[s]) and self.table[s, j] != -1
                       and not 0 <= self.table[s, j] < self.n_pages else x for j, x in enumerate(row)]
            self.table[s, :m] = row
            self.kv_len[s] = sizes[s]
        self.refs = after
        return copies, (left, len(copies))

    def compact(self, most):
        used = [i for i in range(self.n_pages - 1, -1, -1) if self.refs[i]]
        free = [i for i in range(self.n_pages) if not self.refs[i]]
        copies = []
        for a, b in list(zip(used, free))[:most]:
            if b > a:
                break
            copies.append((a, b, self.page))
            self.refs[b], self.refs[a] = self.refs[a], 0
        to = {a: b for a, b, _ in copies}
        for s in range(self.n_seq):
            for j in range(self._pages(self._length(s))):
                self.table[s, j] = to.get(int(self.table[s, j]), self.table[s, j])
        used = np.flatnonzero(self.refs)
        return copies, (int(used[-1]) + 1 if len(used) else 0, len(copies))
