"""Eviction of a damaged table: every row, page and count that the bad entries do not name is as the model says."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import host, say
from test_kv_evict_gpu import Cache, _filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layers,stride,page", [(2, 20, 16), (1, 200, 16), (2, 10, 32)])
def test_bad_entries_reach_nothing(device, gx, layers, stride, page):
    """Missing and out-of-pool pages of sequence 0 among kept rows, holes and movers; sequence 1 is whole; sequence 2 is not listed."""
    rng = np.random.default_rng(stride)
    m = _filled(rng, layers, page, (1, 128), [200, 200, 90], stride, spare=5)
    budget, first, recent = 100, 4, 10
    before = {x: getattr(m, x).copy() for x in ("k", "v", "weight", "position")}
    table, references = [list(t) for t in m.table], list(m.references)
    cache = Cache(gx, m)
    held = -(-200 // page)
    bad = {1: -1, held // 3: -3, held - 1: len(references) + 5, held - 3: 2 ** 31 - 1}
    for column, entry in bad.items():
        cache.table[0, column] = entry
    say("bad entries", layers, stride, page)
    assert cache.evict([0, 1], budget, first, recent) == 0
    # Holes and movers of sequence 0, by the model's rule.
    n, dropped = 200, m.dropped[0]
    last = n + dropped - recent
    stands = [m.position[0, j] < first or m.position[0, j] >= last for j in range(n)]
    kept = set(sorted(range(n), key=lambda j: (not stands[j], -float(m.weight[0, j]), j))[:budget])
    holes, movers = [j for j in range(budget) if j not in kept], sorted(j for j in kept if j >= budget)
    assert len(holes) == len(movers) > 5
    assert m.evict([0, 1], budget, first, recent) == 0
    # Sequence 0: rows whose pages exist moved, the others are as they were; weights and positions moved all the same.
    for pool in ("k", "v"):
        want, old = getattr(m, pool), before[pool]
        for p in table[0]:
            want[:, p] = old[:, p]
        for j, s in zip(holes, movers):
            if j // page not in bad and s // page not in bad:
                want[:, table[0][j // page], j % page] = old[:, table[0][s // page], s % page]
        got = host(getattr(cache, pool))
        assert np.array_equal(got.view(np.int16), want.view(np.int16))
    assert np.array_equal(host(cache.weight).view(np.int32), m.weight.view(np.int32)) and np.array_equal(host(cache.position), m.position)
    assert host(cache.dropped).tolist() == m.dropped and host(cache.lengths).tolist() == m.lengths
    # Pages past the budget are given back where the table still named them.
    need = -(-budget // page)
    want = list(references)
    for column in range(need, held):
        want[table[1][column]] -= 1
        if column not in bad:
            want[table[0][column]] -= 1
    assert host(cache.references).tolist() == want
    expect = m.table_array()
    for column, entry in bad.items():
        if column < need:
            expect[0, column] = entry
    assert np.array_equal(host(cache.table), expect)


def test_positions_that_all_stand(device, gx):
    """Damaged positions that protect more rows than the budget protect none: weights decide, and the rows' moves are the model's."""
    rng = np.random.default_rng(34)
    m = _filled(rng, 2, 16, (1, 128), [150, 200], 20)
    m.position[1] = 0
    cache = Cache(gx, m)
    say("all stand")
    assert m.evict([0, 1], 100, 4, 10) == cache.evict([0, 1], 100, 4, 10) == 0
    cache.check()
