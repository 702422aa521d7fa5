"""Paged key-value cache for generation: host bookkeeping over one pool of pages.

A page holds `page_size` tokens of every head of one layer's keys or values; the same page number is used in all layers.
Sequences list their pages in order.  Forked sequences share full pages; a shared page that is not full is copied when one
of its owners grows (copy on write).  Freed pages are handed out again, lowest number first, and `compact` moves the live
ones to the front of the pool.  All device work is `paged_append_`, `copy_pages_` and `paged_attention`."""
import heapq

import numpy as np

from .. import _C
from ..functional import copy_pages_, paged_append_, paged_attention


class PagedKVCache:
    def __init__(self, num_layers, num_heads, head_dim, num_pages, page_size=16, dtype="float32", device="cpu"):
        for name, value in (("num_layers", num_layers), ("num_heads", num_heads), ("head_dim", head_dim), ("num_pages", num_pages),
                            ("page_size", page_size)):
            if int(value) <= 0:
                raise ValueError(f"PagedKVCache: {name} must be positive")
        self.num_layers, self.num_heads, self.head_dim = int(num_layers), int(num_heads), int(head_dim)
        self.num_pages, self.page_size = int(num_pages), int(page_size)
        self.dtype, self.device = str(dtype), str(device)
        shape = [2 * self.num_layers, self.num_pages, self.num_heads, self.page_size, self.head_dim]
        self.pool = _C._zeros_on(shape, self.dtype, self.device)  # keys of layer i at 2i, its values at 2i + 1
        self._layers = [(self.pool[2 * i], self.pool[2 * i + 1]) for i in range(self.num_layers)]
        self._free = list(range(self.num_pages))  # a heap: lowest page first
        self._owners = [0] * self.num_pages
        self._pages, self._lengths = {}, {}
        self._next = 0

    # ------------------------------------------------------------ bookkeeping
    @property
    def free_pages(self):
        return len(self._free)

    def length(self, sequence):
        return self._lengths[self._known(sequence)]

    def pages(self, sequence):
        return tuple(self._pages[self._known(sequence)])

    def _known(self, sequence):
        if sequence not in self._pages:
            raise KeyError(f"PagedKVCache: no sequence {sequence!r}")
        return sequence

    def _take(self):
        page = heapq.heappop(self._free)
        self._owners[page] = 1
        return page

    def _drop(self, page):
        self._owners[page] -= 1
        if self._owners[page] == 0:
            heapq.heappush(self._free, page)

    def add(self):
        """A new, empty sequence; returns its number."""
        sequence, self._next = self._next, self._next + 1
        self._pages[sequence], self._lengths[sequence] = [], 0
        return sequence

    def extend(self, sequences, counts):
        """Makes room for `counts` more tokens of each sequence (one number for all, or one each) and counts them as there;
        returns the places where they begin.  Raises, with nothing changed, when the free pages do not suffice."""
        return self._extend(sequences, counts)[0]

    def _extend(self, sequences, counts):
        """`extend` that also returns what `_take_back` needs to undo it."""
        sequences = [self._known(s) for s in sequences]
        if len(set(sequences)) != len(sequences):
            raise ValueError("PagedKVCache: a sequence is given twice")
        counts = [int(counts)] * len(sequences) if np.isscalar(counts) else [int(n) for n in counts]
        if len(counts) != len(sequences) or any(n < 0 for n in counts):
            raise ValueError("PagedKVCache: as many counts as sequences, none negative")
        starts = [self._lengths[s] for s in sequences]
        owners = dict()  # owners that shared pages have left once earlier sequences of this call took copies
        private, fresh = [], []
        for s, start, n in zip(sequences, starts, counts):
            pages, last = self._pages[s], start // self.page_size
            copies = False
            if n > 0 and last < len(pages):  # the page that the next token goes to is there already
                page = pages[last]
                left = owners.get(page, self._owners[page])
                copies = left > 1
                if copies:
                    owners[page] = left - 1
            private.append(copies)
            fresh.append(max(0, -(-(start + n) // self.page_size) - len(pages)))
        need = sum(private) + sum(fresh)
        if need > len(self._free):
            raise RuntimeError(f"PagedKVCache: out of pages ({need} needed, {len(self._free)} of {self.num_pages} free)")
        sources, destinations, before = [], [], []
        for s, start, n, copies, more in zip(sequences, starts, counts, private, fresh):
            pages = self._pages[s]
            shared = None
            if copies:
                last = start // self.page_size
                page = self._take()
                shared = pages[last]
                sources.append(shared)
                destinations.append(page)
                self._drop(shared)
                pages[last] = page
            before.append((s, start, len(pages), shared))
            pages.extend(self._take() for _ in range(more))
            self._lengths[s] = start + n
        if sources:
            try:
                copy_pages_(self.pool, sources, destinations, dim=1)
            except BaseException:
                self._take_back(before)
                raise
        return starts, before

    def _take_back(self, before):
        """Undoes an `_extend` behind which nothing else has happened: lengths, page lists and shared pages as before."""
        for s, length, count, shared in reversed(before):
            pages = self._pages[s]
            while len(pages) > count:
                self._drop(pages.pop())
            if shared is not None:
                last = length // self.page_size
                self._drop(pages[last])
                pages[last] = shared
                self._owners[shared] += 1
            self._lengths[s] = length

    def fork(self, sequence):
        """A new sequence with the same tokens; the pages are shared until one of the two grows."""
        pages = self._pages[self._known(sequence)]
        new = self.add()
        for page in pages:
            self._owners[page] += 1
        self._pages[new], self._lengths[new] = list(pages), self._lengths[sequence]
        return new

    def free(self, sequence):
        for page in self._pages.pop(self._known(sequence)):
            self._drop(page)
        del self._lengths[sequence]

    def reorder(self, sequences, parents):
        """Beam search's step: entry i becomes a fork of sequences[parents[i]]; the old sequences are freed."""
        sequences = [self._known(s) for s in sequences]
        if len(set(sequences)) != len(sequences):
            raise ValueError("PagedKVCache: a sequence is given twice")
        parents = [int(p) for p in parents]
        if any(not 0 <= p < len(sequences) for p in parents):
            raise IndexError("PagedKVCache: a parent is out of range")
        chosen = [sequences[p] for p in parents]
        new = [self.fork(s) for s in chosen]
        for s in sequences:
            self.free(s)
        return new

    def compact(self):
        """Moves the live pages to the lowest numbers; returns how many were moved."""
        live = [p for p in range(self.num_pages) if self._owners[p] > 0]
        holes = [p for p in range(len(live)) if self._owners[p] == 0]
        moved = [p for p in live if p >= len(live)]  # as many as there are holes below
        if not moved:
            return 0
        copy_pages_(self.pool, moved, holes, dim=1)
        to = dict(zip(moved, holes))
        for pages in self._pages.values():
            pages[:] = [to.get(p, p) for p in pages]
        for old, new in to.items():
            self._owners[new], self._owners[old] = self._owners[old], 0
        self._free = list(range(len(live), self.num_pages))
        return len(moved)

    # ---------------------------------------------------------------- device
    def _whole(self, values):
        t = _C.from_numpy(np.ascontiguousarray(values, dtype=np.int32))
        return t if self.device == "cpu" else t.to(self.device)

    def table(self, sequences):
        """The page table of some sequences: int32 [B, most pages] on the cache's device."""
        rows = [self._pages[self._known(s)] for s in sequences]
        table = np.zeros((len(rows), max([len(r) for r in rows] + [1])), dtype=np.int32)
        for row, pages in zip(table, rows):
            row[: len(pages)] = pages
        return self._whole(table)

    def lengths(self, sequences):
        """The lengths of some sequences: int32 [B] on the cache's device."""
        return self._whole([self._lengths[self._known(s)] for s in sequences])

    def append(self, layer, k, v, table, starts, counts=None):
        """Writes k / v [B, T, H, D] of one layer from places `starts` on (see `functional.paged_append_`)."""
        paged_append_(*self._layers[layer], k, v, table, starts, counts)

    def attend(self, layer, q, table, lengths, scale=None):
        """Attention of q [B, H, D] over the first `lengths` tokens in one layer (see `functional.paged_attention`)."""
        return paged_attention(q, *self._layers[layer], table, lengths, scale)
