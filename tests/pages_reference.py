"""A book of pages stated plainly: lists, one step after the other."""


class Book:
    def __init__(self, sequences, width, pages, page_tokens):
        self.width, self.page = width, page_tokens
        self.table = [[-1] * width for _ in range(sequences)]
        self.lengths, self.refs = [0] * sequences, [0] * pages
        self.report = [0, 0, 0, 0]

    def _pages_of(self, tokens):
        return -(-tokens // self.page)

    def _free(self):
        return [i for i, n in enumerate(self.refs) if n == 0]

    def grow(self, news):
        wanted = [n + max(m, 0) for n, m in zip(self.lengths, news)]
        if any(n > self.width * self.page for n in wanted):
            self.report = [-1, 0, 0, 0]
            return
        need = sum(self._pages_of(w) - self._pages_of(n) for w, n in zip(wanted, self.lengths))
        free = self._free()
        if need > len(free):
            self.report = [need - len(free), 0, 0, 0]
            return
        for b, w in enumerate(wanted):
            for i in range(self._pages_of(self.lengths[b]), self._pages_of(w)):
                page = free.pop(0)
                self.table[b][i], self.refs[page] = page, 1
            self.lengths[b] = w
        self.report = [0, need, 0, 0]

    def fork(self, parents, keep=None):
        """Returns the pairs."""
        n_seq = len(self.table)
        none = [[-1, -1]] * n_seq
        if any(p >= n_seq for p in parents):
            self.report = [-1, 0, 0, 0]
            return none
        old = [self.table[b][:self._pages_of(self.lengths[b])] for b in range(n_seq)]
        new = [0 if p < 0 else min(self.lengths[p], max(keep[b], 0) if keep else 1 << 40) for b, p in enumerate(parents)]
        rows = [[] if p < 0 else old[p][:self._pages_of(new[b])] for b, p in enumerate(parents)]
        stays = [p == b and new[b] == self.lengths[b] for b, p in enumerate(parents)]
        # who has a name for what, before anybody takes a last page that is not full
        tails = [not s and bool(n % self.page) for s, n in zip(stays, new)]
        names = list(self.refs)  # (what rows do not account for is somebody else's)
        for row in old:
            for page in row:
                names[page] -= 1
        for b in range(n_seq):
            for page in rows[b][:len(rows[b]) - tails[b]]:
                names[page] += 1
        needing = []
        for b in range(n_seq):
            if tails[b]:
                page = rows[b][-1]
                if names[page] == 0:
                    names[page] = 1
                    continue
                needing.append(b)
        # (those that need a page look for it when every page that somebody continues in has its name)
        free = [i for i, n in enumerate(names) if n == 0]
        if len(needing) > len(free):
            self.report = [len(needing) - len(free), 0, 0, 0]
            return none
        pairs = []
        for b in needing:
            page = free.pop(0)
            pairs.append([rows[b][-1], page])
            rows[b][-1], names[page] = page, 1
        self.refs, self.lengths = names, new
        self.table = [r + [-1] * (self.width - len(r)) for r in rows]
        self.report = [0, len(needing), len(needing), 0]
        return pairs + none[len(pairs):]

    def compact(self):
        """Returns the pairs."""
        used = sum(n > 0 for n in self.refs)
        holes = [i for i in range(used) if self.refs[i] == 0]
        moves = [i for i in range(used, len(self.refs)) if self.refs[i] > 0]
        to = dict(zip(moves, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        self.report = [0, used, len(holes), 0]
        return [[a, b] for a, b in to.items()] + [[-1, -1]] * (len(self.refs) - len(to))

    def check(self):
        """The rules that every call keeps."""
        count = [0] * len(self.refs)
        for row, n in zip(self.table, self.lengths):
            held = self._pages_of(n)
            assert all(p >= 0 for p in row[:held]) and all(p == -1 for p in row[held:])
            for p in row[:held]:
                count[p] += 1
        assert count == self.refs
        for row, n in zip(self.table, self.lengths):
            if n % self.page:
                assert count[row[n // self.page]] == 1
