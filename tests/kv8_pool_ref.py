"""The pool's operators on lists, one entry at a time."""


def used(n, page):
    return -(-n // page)


def clamp(n, W, page):
    return min(max(n, 0), W * page)


class Pool:
    """refs, and pages[p]: any value that stands for what page p holds."""

    def __init__(self, P, page):
        self.P, self.page, self.refs, self.pages = P, page, [0] * P, [("page", p) for p in range(P)]

    def is_page(self, p):
        return 0 <= p < self.P

    def fork(self, table, lens, parents, release):
        W = len(table[0])
        rows, new_lens = [], []
        for p in parents:
            n = clamp(lens[p], W, self.page) if 0 <= p < len(table) else 0
            row = [table[p][j] if j < used(n, self.page) else -1 for j in range(W)]
            for e in row[:used(n, self.page)]:
                if self.is_page(e):
                    self.refs[e] += 1
            rows.append(row)
            new_lens.append(n)
        if release:
            for b, row in enumerate(table):
                for e in row[:used(clamp(lens[b], W, self.page), self.page)]:
                    if self.is_page(e):
                        self.refs[e] -= 1
        return rows, new_lens

    def resize(self, table, lens, new_lens):
        W = len(table[0])
        lens, new_lens = [clamp(n, W, self.page) for n in lens], [clamp(n, W, self.page) for n in new_lens]
        for row, a, b in zip(table, lens, new_lens):
            for j in range(used(b, self.page), used(a, self.page)):
                if self.is_page(row[j]):
                    self.refs[row[j]] -= 1
                    row[j] = -1
        slots = []
        for i, (row, a, b) in enumerate(zip(table, lens, new_lens)):
            if b <= a:
                continue
            j = used(a, self.page)
            if a % self.page and self.is_page(row[j - 1]) and self.refs[row[j - 1]] > 1:
                slots.append((i, j - 1, row[j - 1]))
            slots += [(i, k, None) for k in range(j, used(b, self.page))]
        free = [p for p in range(self.P) if self.refs[p] <= 0]
        if len(slots) > len(free):
            return len(slots) - len(free)
        held = list(self.pages)
        for p, (i, j, copied) in zip(free, slots):
            if copied is not None:
                self.refs[copied] -= 1
                self.pages[p] = held[copied]
            table[i][j] = p
            self.refs[p] = 1
        return 0

    def compact(self, *tables):
        live = [p for p in range(self.P) if self.refs[p] > 0]
        n = len(live)
        names = dict(zip([p for p in live if p >= n], [p for p in range(n) if self.refs[p] <= 0]))
        for a, b in names.items():
            self.pages[b] = self.pages[a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        for t in tables:
            for row in t:
                row[:] = [names.get(e, e) for e in row]
        return n
