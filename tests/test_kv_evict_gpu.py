"""Eviction of a paged K/V cache to a budget on the GPU against a plain model with lists: state and rows, bit for bit."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import dev, empty, host, say
from kv_pages_model import PagesModel

pytestmark = pytest.mark.gpu


class Bounded(PagesModel):
    """The pages' model with weight, position and dropped beside it."""

    def __init__(self, layers, pages, page, kv_heads, d, sequences, stride, rng):
        super().__init__(layers, pages, page, kv_heads, d, sequences, stride, rng)
        self.weight = np.full((sequences, stride * page), 9.0, np.float32)
        self.position = np.full((sequences, stride * page), -7, np.int32)
        self.dropped = [0] * sequences

    def begin(self, sequences, tokens):
        for s, t in zip(sequences, tokens):
            n = self.lengths[s]
            self.dropped[s] = self.dropped[s] if n else 0
            for j in range(n, min(n + t, self.stride * self.page)):
                self.weight[s, j], self.position[s, j] = 0, j + self.dropped[s]

    def evict(self, sequences, budget, first, recent):
        before, free, plans = list(self.references), self._free_pages(), []
        for s in sequences:
            n = self.lengths[s]
            if n <= budget:
                continue
            last = n + self.dropped[s] - recent
            value = [np.inf if np.isnan(x) else x + 0.0 for x in self.weight[s, :n].tolist()]
            nan = np.isnan(self.weight[s, :n])
            stands = [self.position[s, j] < first or self.position[s, j] >= last for j in range(n)]
            order = sorted(range(n), key=lambda j: (not stands[j], not nan[j], -value[j], j))
            kept = sorted(order[:budget])
            below = set(kept)
            holes, movers = [j for j in range(budget) if j not in below], [j for j in kept if j >= budget]
            columns = [c for c in sorted({j // self.page for j in holes}) if before[self.table[s][c]] > 1]
            plans.append((s, n, kept, holes, movers, columns))
        if sum(len(p[-1]) for p in plans) > len(free):
            return 1
        for s, n, kept, holes, movers, columns in plans:
            old = list(self.table[s])
            for c in columns:
                to = free.pop(0)
                self.references[old[c]] -= 1
                self.references[to] = 1
                self.table[s][c] = to
                for j in kept:
                    if j // self.page == c and j < budget:
                        self.k[:, to, j % self.page] = self.k[:, old[c], j % self.page]
                        self.v[:, to, j % self.page] = self.v[:, old[c], j % self.page]
            for j, m in zip(holes, movers):
                for pool in (self.k, self.v):
                    pool[:, self.table[s][j // self.page], j % self.page] = pool[:, old[m // self.page], m % self.page]
                self.weight[s, j], self.position[s, j] = self.weight[s, m], self.position[s, m]
            for c in range(self._need(budget), len(old)):
                self.references[old[c]] -= 1
            self.table[s] = self.table[s][:self._need(budget)]
            self.dropped[s] += n - budget
            self.lengths[s] = budget
        return 0


class Cache:
    """The model and the device side, made alike."""

    def __init__(self, gx, model):
        self.gx, self.model = gx, model
        m = model
        self.k, self.v = dev(m.k), dev(m.v)
        self.table, self.lengths = dev(m.table_array()), dev(np.array(m.lengths, np.int32))
        self.references = dev(np.array(m.references, np.int32))
        self.weight, self.position, self.dropped = dev(m.weight), dev(m.position), dev(np.array(m.dropped, np.int32))
        self.pages = gx.KvPages.of(self.k, self.v, self.table, self.lengths, self.references)
        self.weights = gx.KvWeights.of(self.pages, self.weight, self.position, self.dropped)
        self.status = empty((1,), np.int32)

    def workspace(self, count, budget):
        import torch
        return torch.full((gx_bytes(self.gx, self.pages, count, budget),), 0xff, dtype=torch.uint8, device="cuda")

    def evict(self, sequences, budget, first, recent, stream=None):
        self.gx.launch_kv_pages_evict(self.pages, self.weights, sequences, budget, first, recent, self.status,
                                      self.workspace(len(sequences), budget), stream=stream)
        return int(host(self.status)[0])

    def check(self):
        m = self.model
        for got, want in ((self.table, m.table_array()), (self.lengths, m.lengths), (self.references, m.references), (self.dropped, m.dropped),
                          (self.position, m.position), (self.weight.view(dtype=self.position.dtype), m.weight.view(np.int32)),
                          (self.k.view(dtype=self.k.new_empty(0, dtype=self.k.dtype).dtype), m.k), (self.v, m.v)):
            assert np.array_equal(host(got), np.array(want), equal_nan=False) if host(got).dtype.kind != "f" else \
                np.array_equal(host(got).view(np.int16), np.array(want).view(np.int16))


def gx_bytes(gx, pages, count, budget):
    return max(16, gx.kv_pages_evict_workspace_bytes(pages, count, budget))


def _filled(rng, layers, page, heads, lengths, stride, spare=6, shared=0):
    """Sequences of these lengths (the first `shared` tokens on common pages), weights of earlier steps, positions with gaps."""
    kv_heads, d = heads
    m = Bounded(layers, sum(-(-n // page) for n in lengths) + spare, page, kv_heads, d, len(lengths) + 1, stride, rng)
    order = rng.permutation(len(m.references)).tolist()
    common = [order.pop() for _ in range(shared // page)]
    for s, n in enumerate(lengths):
        mine = (common if n >= shared else []) + []
        while len(mine) * page < n:
            mine.append(order.pop())
        m.table[s], m.lengths[s], m.dropped[s] = mine, n, int(rng.integers(0, 50))
        for p in mine:
            m.references[p] += 1
        m.position[s, :n] = rng.permutation(rng.choice(n + m.dropped[s], n, replace=False))
        m.weight[s, :n] = rng.random(n) ** 8 * 5
    return m


@pytest.mark.parametrize("layers,page,heads,lengths,budget,first,recent,shared", [
    (1, 16, (1, 128), [2], 1, 0, 0, 0),                        # down to one row
    (1, 16, (1, 128), [17, 16, 15, 0], 16, 1, 1, 0),           # at, above and below the budget
    (2, 16, (2, 128), [100, 37, 64], 37, 4, 8, 0),
    (1, 16, (1, 256), [48, 33], 16, 8, 8, 0),                  # nothing but what stays for its position
    (1, 32, (3, 128), [200, 90], 50, 0, 0, 0),
    (2, 64, (1, 256), [1500, 1100, 1030], 1024, 16, 100, 0),
    (1, 16, (1, 128), [5000, 4099], 4097, 0, 4097, 0),
    (2, 16, (1, 128), [80, 70, 90, 20], 50, 2, 5, 48),         # shared pages: private copies
    (1, 32, (1, 128), [130, 130], 100, 0, 0, 128),             # both holders leave the same pages
    (1, 4096, (1, 128), [9000], 4100, 3, 10, 0),
    (1, 16, (1, 128), [70000], 30000, 10, 1000, 0),
])
def test_eviction_equals_the_model(device, gx, layers, page, heads, lengths, budget, first, recent, shared):
    rng = np.random.default_rng(budget + page + len(lengths))
    m = _filled(rng, layers, page, heads, lengths, -(-max(lengths) // page) + 2, spare=40 if shared else 3, shared=shared)
    cache = Cache(gx, m)
    say("eviction", layers, page, heads, lengths, budget, first, recent, shared)
    sequences = rng.permutation(len(lengths)).tolist()
    assert m.evict(sequences, budget, first, recent) == 0
    assert cache.evict(sequences, budget, first, recent) == 0
    cache.check()
    assert m.evict(sequences, budget, first, recent) == cache.evict(sequences, budget, first, recent) == 0
    cache.check()                                              # nothing is left to do


@pytest.mark.parametrize("page,lengths,stride,budget,shared", [
    (16, [100, 37, 64, 50, 38, 90, 0, 200], 16, 37, 0),        # more sequences than one workgroup chooses for
    (16, [120, 37, 1000, 90], 64, 40, 0), (16, [120, 37, 90], 70, 40, 32), (16, [90, 800], 64, 700, 32)])
def test_tables_of_many_sizes(device, gx, page, lengths, stride, budget, shared):
    rng = np.random.default_rng(budget + stride)
    m = _filled(rng, 2, page, (1, 128), lengths, stride, spare=20, shared=shared)
    cache = Cache(gx, m)
    say("tables of many sizes", lengths, stride, budget, shared)
    for _ in range(2):                                         # the second time there is nothing to do
        sequences = rng.permutation(len(lengths)).tolist()
        assert m.evict(sequences, budget, 3, 9) == 0
        assert cache.evict(sequences, budget, 3, 9) == 0
        cache.check()


def test_ties_zeros_infinities_and_nan(device, gx):
    rng = np.random.default_rng(31)
    for values in ([0.0], [-0.0, 0.0], [1.0, 1.0, 2.0], [np.nan, 1.0, np.inf], [np.nan], [np.inf, -np.inf, -1.0], [1e-45, 0.0, 2e-45],
                   [-1.0, -2.0, -0.5]):
        m = _filled(rng, 1, 16, (1, 128), [300, 1500], 100)
        for s, n in enumerate((300, 1500)):
            m.weight[s, :n] = rng.choice(np.array(values, np.float32), n)
        cache = Cache(gx, m)
        say("ties", values)
        assert m.evict([0, 1], 130, 3, 20) == cache.evict([0, 1], 130, 3, 20) == 0
        cache.check()


def test_too_few_pages_change_nothing(device, gx):
    rng = np.random.default_rng(32)
    m = _filled(rng, 1, 16, (1, 128), [96, 96, 96], 8, spare=2 - 12 + 2, shared=96)
    cache = Cache(gx, m)
    say("too few pages")
    assert m.evict([0, 1, 2], 40, 0, 0) == cache.evict([0, 1, 2], 40, 0, 0) == 1
    cache.check()
    # A sequence whose pages are its own needs no copy and is not held up.
    m = _filled(rng, 1, 16, (1, 128), [96], 8, spare=0)
    cache = Cache(gx, m)
    assert m.evict([0], 40, 0, 0) == cache.evict([0], 40, 0, 0) == 0
    cache.check()


def test_pages_reserved_past_the_length_go_back(device, gx):
    rng = np.random.default_rng(33)
    m = _filled(rng, 1, 16, (1, 128), [100, 30], 40, spare=10)
    for s in (0, 1):
        for _ in range(3):
            p = m._free_pages()[0]
            m.table[s].append(p)
            m.references[p] = 1
    cache = Cache(gx, m)
    say("reserved pages")
    assert m.evict([0, 1], 50, 0, 0) == cache.evict([0, 1], 50, 0, 0) == 0
    cache.check()


def test_missing_pages_and_damaged_state_stay_in_bounds(device, gx):
    """Rows without a page are passed over; positions that say that everything stays do not lead past the budget."""
    rng = np.random.default_rng(34)
    m = _filled(rng, 1, 16, (1, 128), [200, 200], 20)
    cache = Cache(gx, m)
    cache.table[0, 3], cache.table[0, 11], cache.table[0, 5] = -1, len(m.references) + 5, -3
    cache.position[1] = 0                                      # all "first"
    say("damaged state")
    assert cache.evict([0, 1], 100, 4, 10) == 0
    assert host(cache.lengths)[:2].tolist() == [100, 100]
    order = sorted(range(200), key=lambda j: (-m.weight[1, j], j))[:100]
    assert sorted(host(cache.weight)[1, :100].tolist()) == sorted(m.weight[1, order].tolist())


def test_begin(device, gx):
    rng = np.random.default_rng(35)
    m = _filled(rng, 1, 16, (1, 128), [100, 0, 158, 40], 10)
    m.dropped[1] = 77                                          # of what the slot held before
    cache = Cache(gx, m)
    say("begin")
    for tokens in ([3, 9, 5, 0], [0, 160, 1, 20], [300, 1, 2, 1]):
        m.begin([0, 1, 2, 3], tokens)
        gx.launch_kv_weights_begin(cache.pages, cache.weights, [0, 1, 2, 3], tokens)
        cache.check()


@pytest.mark.parametrize("page", [16, 64])
def test_steps_in_a_graph(device, gx, page):
    """reserve, begin, advance and evict recorded once; every replay drops as many rows as it takes."""
    import torch
    rng = np.random.default_rng(36)
    budget, tokens = 5 * page - 3, page // 2 + 1
    m = _filled(rng, 1, page, (2, 128), [budget, budget - 20, 3], 8, spare=12)
    cache = Cache(gx, m)
    work = torch.empty(max(gx.kv_pages_workspace_bytes(cache.pages), gx_bytes(gx, cache.pages, 3, budget)), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph, listed = torch.cuda.CUDAGraph(), [0, 1, 2]
    with torch.cuda.graph(graph, stream=stream):
        gx.launch_kv_pages_reserve(cache.pages, listed, tokens, cache.status, work)
        gx.launch_kv_weights_begin(cache.pages, cache.weights, listed, [tokens] * 3)
        gx.launch_kv_pages_advance(cache.pages, listed, tokens)
        gx.launch_kv_pages_evict(cache.pages, cache.weights, listed, budget, 4, page, cache.status, work)
    say("steps in a graph", page)
    for _ in range(6):
        assert m.reserve(listed, tokens) == 0
        m.begin(listed, [tokens] * 3)
        m.advance(listed, tokens)
        assert m.evict(listed, budget, 4, page) == 0
        graph.replay()
        torch.cuda.synchronize()
        cache.check()
        # Eager work between the replays: the rows get weights, as attention gives them.
        add = (rng.random(m.weight.shape) * 0.1).astype(np.float32)
        m.weight += add
        cache.weight += dev(add)
