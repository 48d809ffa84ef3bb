"""Budgets that no sequence reaches: nothing changes, and the call takes no longer than any other."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import say
from test_kv_evict_gpu import Cache, _filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths,stride", [([100, 37], 16), ([100, 37, 64, 200, 90], 16), ([100, 1500], 128)])
@pytest.mark.parametrize("budget", [5000, 1 << 20, (1 << 31) + 5, (1 << 32) - 1])
def test_a_budget_that_no_sequence_reaches(device, gx, lengths, stride, budget):
    """The choice of rows went through the pages of the budget, 2^28 of them, not through those of the table."""
    import torch
    m = _filled(np.random.default_rng(len(lengths)), 1, 16, (1, 128), lengths, stride)
    cache = Cache(gx, m)
    say("large budget", lengths, stride, budget)
    listed = list(range(len(lengths)))
    assert cache.evict(listed, 5000, 3, 9) == 0               # (first calls load code)
    work = cache.workspace(len(listed), budget)
    began, ended = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    began.record()
    gx.launch_kv_pages_evict(cache.pages, cache.weights, listed, budget, 3, budget - 3, cache.status, work)
    ended.record()
    torch.cuda.synchronize()
    assert int(cache.status.cpu()[0]) == 0
    cache.check()
    assert began.elapsed_time(ended) < 20                     # ms; a call takes 0.04
