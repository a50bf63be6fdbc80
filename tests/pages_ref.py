"""The page calls done one step after the other, on lists: the reference of the device's
page bookkeeping (prichs_kv_pages_*)."""
import numpy as np

PAGE = 64


class Pages:
    def __init__(self, refs, table, lens=None, data=None):
        self.refs, self.table = [int(r) for r in refs], [[int(p) for p in row] for row in table]
        self.width = len(self.table[0]) if self.table else 0
        self.lens = None if lens is None else [int(n) for n in lens]
        self.data = None if data is None else np.array(data)

    def names(self, p):
        return 0 <= p < len(self.refs)

    def take(self, n):
        """The n lowest free pages, -1 for those that are missing, and how many are."""
        free = [p for p, r in enumerate(self.refs) if r <= 0][:n]
        for p in free:
            self.refs[p] = 1
        return free + [-1] * (n - len(free)), n - len(free)

    def reserve(self, counts):
        at, beyond = [], 0
        for b, n in enumerate(counts):
            if n <= 0:
                continue
            first = max(self.lens[b], 0)
            for e in range(first // PAGE, (first + n - 1) // PAGE + 1):
                if e >= self.width:
                    beyond += 1
                elif not self.names(self.table[b][e]):
                    at.append((b, e))
        pages, short = self.take(len(at))
        for (b, e), p in zip(at, pages):
            self.table[b][e] = p
        return short + beyond

    def fork(self, parents, children):
        rows = range(len(self.table))
        used, items = set(), []
        for p, c in zip(parents, children):
            if c in rows and c not in used:
                used.add(c)
                items.append((p, c))
        items = [(p, c) for p, c in items if p in rows and p not in used]
        want = []
        for p, c in items:
            L = min(max(self.lens[p], 0), self.width * PAGE)
            part = self.table[p][L // PAGE] if L % PAGE else -1
            want.append(self.names(part))
        pages, short = self.take(sum(want))
        for (p, c), w in zip(items, want):
            L = min(max(self.lens[p], 0), self.width * PAGE)
            full = L // PAGE
            row = [q if self.names(q) else -1 for q in self.table[p][:full]]
            for q in row:
                if q >= 0:
                    self.refs[q] += 1
            if L % PAGE:
                new = pages.pop(0) if w else -1
                if new >= 0 and self.data is not None:
                    self.data[new] = self.data[self.table[p][full]]
                row.append(new)
            self.table[c] = row + [-1] * (self.width - len(row))
            self.lens[c] = L
        return short

    def release(self, rows, keep=None):
        for i, b in enumerate(rows):
            if not 0 <= b < len(self.table):
                continue
            first = 0 if keep is None else -(-max(keep[i], 0) // PAGE)
            for e in range(first, self.width):
                p = self.table[b][e]
                if self.names(p) and self.refs[p] > 0:
                    self.refs[p] -= 1
                self.table[b][e] = -1

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r > 0]
        new = [p if r > 0 else -1 for p, r in enumerate(self.refs)]
        holes = [p for p, r in enumerate(self.refs) if r <= 0 and p < len(live)]
        for dst, src in zip(holes, [p for p in live if p >= len(live)]):
            new[src] = dst
            self.refs[dst], self.refs[src] = self.refs[src], 0
            if self.data is not None:
                self.data[dst] = self.data[src]
        self.table = [[new[p] if self.names(p) else p for p in row] for row in self.table]
        return len(live), new
