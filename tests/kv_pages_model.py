"""A plain model of the paged K/V cache: Python lists for the state, numpy for the pools, one step after another."""
from __future__ import annotations

import numpy as np


class PagesModel:
    def __init__(self, layers, pages, page_tokens, kv_heads, head_size, sequences, stride, rng):
        self.page, self.stride = page_tokens, stride
        shape = (layers, pages, page_tokens, kv_heads, head_size)
        self.k = rng.standard_normal(shape).astype(np.float16)
        self.v = rng.standard_normal(shape).astype(np.float16)
        self.table = [[] for _ in range(sequences)]
        self.lengths = [0] * sequences
        self.references = [0] * pages

    def _free_pages(self):
        return [p for p, n in enumerate(self.references) if n == 0]

    def _need(self, tokens):
        return -(-tokens // self.page)

    def fork(self, parent, children):
        shared = self.table[parent][:self._need(self.lengths[parent])]
        for c in children:
            self.free([c])
            self.table[c] = list(shared)
            self.lengths[c] = self.lengths[parent]
            for p in shared:
                self.references[p] += 1

    def free(self, sequences, keep=None):
        for i, s in enumerate(sequences):
            self.lengths[s] = min(self.lengths[s], keep[i] if keep else 0)
            held = self._need(self.lengths[s])
            for p in self.table[s][held:]:
                self.references[p] -= 1
            self.table[s] = self.table[s][:held]

    def reserve(self, sequences, tokens):
        """Returns the status.  A shared tail is copied unless every other holder has just copied it."""
        asked = []
        for i, s in enumerate(sequences):
            n = self.lengths[s]
            if self._need(n + tokens) > self.stride:
                return 1
            tail = self.table[s][n // self.page] if n % self.page else None
            copies = False
            if tail is not None:
                requests = [j for j, o in enumerate(sequences)
                            if self.lengths[o] % self.page and self.table[o][self.lengths[o] // self.page] == tail]
                holders = self.references[tail]
                copies = holders > 1 and (len(requests) < holders or i != requests[-1])
            asked.append((s, tail, copies, max(0, self._need(n + tokens) - len(self.table[s]))))
        free = self._free_pages()
        if sum(c + n for _, _, c, n in asked) > len(free):
            return 1
        for s, tail, copies, new in asked:
            if copies:
                to, rows = free.pop(0), self.lengths[s] % self.page
                self.k[:, to, :rows] = self.k[:, tail, :rows]
                self.v[:, to, :rows] = self.v[:, tail, :rows]
                self.references[tail] -= 1
                self.references[to] = 1
                self.table[s][self.lengths[s] // self.page] = to
            for _ in range(new):
                to = free.pop(0)
                self.references[to] = 1
                self.table[s].append(to)
        return 0

    def append(self, layer, key, value, sequences):
        for i, s in enumerate(sequences):
            for t in range(key.shape[1]):
                at = self.lengths[s] + t
                if at // self.page < len(self.table[s]) and self.references[self.table[s][at // self.page]] <= 1:
                    self.k[layer, self.table[s][at // self.page], at % self.page] = key[i, t]
                    self.v[layer, self.table[s][at // self.page], at % self.page] = value[i, t].astype(np.float16)

    def advance(self, sequences, tokens, counts=None):
        for i, s in enumerate(sequences):
            self.lengths[s] = min(self.lengths[s] + (min(counts[i], tokens) if counts is not None else tokens),
                                  self.stride * self.page)

    def copy(self, sources, destinations):
        for a, b in zip(sources, destinations):
            self.k[:, b] = self.k[:, a]
            self.v[:, b] = self.v[:, a]

    def compact(self):
        used = [p for p, n in enumerate(self.references) if n]
        live = len(used)
        movers = [p for p in used if p >= live]
        holes = [p for p in range(live) if self.references[p] == 0]
        to = dict(zip(movers, holes))
        self.copy(movers, holes)
        for a, b in to.items():
            self.references[b], self.references[a] = self.references[a], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return live

    def rows(self, layer, s, count):
        """K and V [count, kv_heads, head_size] of the sequence's first positions, in 64 bits."""
        at = [(self.table[s][i // self.page], i % self.page) for i in range(count)]
        pages, places = [a for a, _ in at], [b for _, b in at]
        return self.k[layer, pages, places].astype(np.float64), self.v[layer, pages, places].astype(np.float64)

    def table_array(self):
        return np.array([row + [-1] * (self.stride - len(row)) for row in self.table], dtype=np.int32)
