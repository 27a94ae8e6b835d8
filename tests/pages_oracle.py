"""The book of a paged cache's pages, entry by entry, and a program that uses one: plain Python over numpy arrays."""
import numpy as np

BAD_PAGE, BAD_BOUND, BAD_SLOT, NO_PAGE = 16, 32, 64, 128


class Book:
    def __init__(self, pages, page_size, slots, max_pages):
        self.page = page_size
        self.refs = np.zeros(pages, np.int32)
        self.tables = np.full((slots, max_pages), -1, np.int32)
        self.lengths = np.zeros(slots, np.int32)
        self.status = 0

    def held(self, n):
        return -(-int(n) // self.page)

    def _lowest(self, n):
        """The n lowest free pages, or None; once an entry of a call has gone without, those behind it do too."""
        if n == 0:
            return []
        free = np.flatnonzero(self.refs == 0)
        if self.short or len(free) < n:
            self.short = True
            self.status |= NO_PAGE
            return None
        return free[:n].tolist()

    def _take(self, slot, first, pages):
        for c, p in enumerate(pages):
            self.tables[slot, first + c] = p
            self.refs[p] = 1

    def grow(self, slots, add):
        self.short, named = False, set()
        for slot, n in zip(slots, add):
            if slot < 0:
                continue
            if slot >= len(self.lengths) or slot in named:
                self.status |= BAD_SLOT
                continue
            named.add(slot)
            if n < 0 or self.lengths[slot] + n > self.tables.shape[1] * self.page:
                self.status |= BAD_BOUND
                continue
            first = self.held(self.lengths[slot])
            pages = self._lowest(self.held(self.lengths[slot] + n) - first)
            if pages is not None:
                self._take(slot, first, pages)
                self.lengths[slot] += n

    def fork(self, parents, children, at=None, copy=lambda source, target: None):
        self.short, named, lengths = False, set(), self.lengths.copy()
        for e, (parent, child) in enumerate(zip(parents, children)):
            if child < 0:
                continue
            if child >= len(lengths) or child in named:
                self.status |= BAD_SLOT
                continue
            named.add(child)
            if not 0 <= parent < len(lengths) or lengths[child] != 0:
                self.status |= BAD_SLOT
                continue
            n = int(lengths[parent]) if at is None else max(0, min(int(lengths[parent]), int(at[e])))
            whole = n // self.page
            pages = self._lowest(self.held(n) - whole)
            if pages is None:
                continue
            self.tables[child] = -1
            self.tables[child, :whole] = self.tables[parent, :whole]
            self.refs[self.tables[parent, :whole]] += 1
            self._take(child, whole, pages)
            for p in pages:
                copy(int(self.tables[parent, whole]), p)
            self.lengths[child] = n

    def free(self, slots):
        for slot in slots:
            if slot < 0:
                continue
            if slot >= len(self.lengths):
                self.status |= BAD_SLOT
                continue
            for c in range(self.held(self.lengths[slot])):
                self.refs[self.tables[slot, c]] -= 1
                self.tables[slot, c] = -1
            self.lengths[slot] = 0

    def compact(self, copy=lambda source, target: None):
        live = np.flatnonzero(self.refs)
        movers, holes = live[live >= len(live)], np.flatnonzero(self.refs[:len(live)] == 0)
        moved = np.where(self.refs > 0, np.arange(len(self.refs)), -1).astype(np.int32)
        for source, target in zip(movers, holes):
            copy(int(source), int(target))
            moved[source] = target
            self.refs[target], self.refs[source] = self.refs[source], 0
        for s, n in enumerate(self.lengths):
            for c in range(self.held(n)):
                self.tables[s, c] = moved[self.tables[s, c]]
        return moved
