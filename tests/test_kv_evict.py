"""CPU tests of chunk attention, attention weights and eviction: what they refuse, before anything is launched."""
from __future__ import annotations

import ctypes

import pytest

from test_kv_pages import _aligned, _ids, cache  # noqa: F401  (the fixture)

BIG = 1 << 20


@pytest.fixture()
def weights(gx):
    arrays = [_aligned(4 * 4 * 48), _aligned(4 * 4 * 48), _aligned(16)]
    w = gx.KvWeights(*(a.ctypes.data for a in arrays))
    w.tensors = arrays
    return w


def _at(x):
    return x if x is None or isinstance(x, int) else x.ctypes.data


def _ref(x):
    return None if x is None else ctypes.byref(x)


def _attention(gx, pages, **change):
    a = dict(layer=0, query=_aligned(1 << 16), gate=_aligned(1 << 16), output=_aligned(1 << 16), sums=_aligned(4096), ids=_ids(0, 1),
             tokens=_ids(1, 2), count=2, q_heads=4, workspace=_aligned(BIG), bytes=BIG)
    a.update(change)
    return gx.lib().gfxinfer_launch_kv_pages_chunk_attention(
        _ref(pages), a["layer"], _at(a["query"]), _at(a["gate"]), _at(a["output"]), _at(a["sums"]), a["ids"], a["tokens"], a["count"],
        a["q_heads"], _at(a["workspace"]), a["bytes"], None)


def _add(gx, pages, weights, **change):
    a = dict(layer=0, query=_aligned(1 << 16), sums=_aligned(4096), ids=_ids(0, 1), tokens=_ids(1, 2), count=2, q_heads=4,
             workspace=_aligned(BIG), bytes=BIG)
    a.update(change)
    return gx.lib().gfxinfer_launch_kv_weights_add(_ref(pages), _ref(weights), a["layer"], _at(a["query"]), _at(a["sums"]), a["ids"],
                                                   a["tokens"], a["count"], a["q_heads"], _at(a["workspace"]), a["bytes"], None)


def _evict(gx, pages, weights, **change):
    a = dict(ids=_ids(0, 1), count=2, budget=20, first=2, recent=3, status=_aligned(16), workspace=_aligned(BIG), bytes=BIG)
    a.update(change)
    return gx.lib().gfxinfer_launch_kv_pages_evict(_ref(pages), _ref(weights), a["ids"], a["count"], a["budget"], a["first"], a["recent"],
                                                   _at(a["status"]), _at(a["workspace"]), a["bytes"], None)


SHARED = [dict(count=0), dict(count=257), dict(ids=_ids(0, 4)), dict(ids=None, count=5), dict(tokens=None), dict(tokens=_ids(0, 0)),
          dict(tokens=_ids(1 << 20, 1)), dict(tokens=_ids(0xffffffff, 0xffffffff))]


@pytest.mark.parametrize("change", SHARED + [
    dict(layer=2), dict(query=None), dict(output=None), dict(q_heads=0), dict(q_heads=3), dict(q_heads=1026), dict(workspace=None),
    dict(bytes=100), dict(query=_aligned(4096).ctypes.data + 2), dict(gate=_aligned(4096).ctypes.data + 8),
    dict(output=_aligned(4096).ctypes.data + 4), dict(sums=_aligned(4096).ctypes.data + 2),
    dict(workspace=_aligned(4096).ctypes.data + 8)])
def test_bad_attention_is_refused(gx, cache, change):  # noqa: F811
    # A wide table, so that positions are divided and the workspace matters.
    cache.table_stride = 1024
    assert _attention(gx, cache, **change) == gx.INVALID_ARGUMENT
    assert gx.last_error()


@pytest.mark.parametrize("change", SHARED + [
    dict(layer=2), dict(query=None), dict(sums=None), dict(q_heads=0), dict(q_heads=3), dict(workspace=None), dict(bytes=8),
    dict(query=_aligned(4096).ctypes.data + 2), dict(sums=_aligned(4096).ctypes.data + 2), dict(ids=_ids(1, 1)),
    dict(workspace=_aligned(4096).ctypes.data + 8)])
def test_bad_weights_are_refused(gx, cache, weights, change):  # noqa: F811
    assert _add(gx, cache, weights, **change) == gx.INVALID_ARGUMENT
    assert gx.last_error()


@pytest.mark.parametrize("change", [
    dict(count=0), dict(count=513), dict(ids=_ids(0, 4)), dict(ids=_ids(1, 1)), dict(ids=None, count=5), dict(budget=0, first=0, recent=0),
    dict(first=18), dict(recent=0xffffffff), dict(status=None), dict(workspace=None), dict(bytes=16),
    dict(workspace=_aligned(4096).ctypes.data + 8)])
def test_bad_evictions_are_refused(gx, cache, weights, change):  # noqa: F811
    assert _evict(gx, cache, weights, **change) == gx.INVALID_ARGUMENT
    assert gx.last_error()


def test_missing_descriptions_are_refused(gx, cache, weights):  # noqa: F811
    assert _attention(gx, None) == _add(gx, None, weights) == _evict(gx, None, weights) == gx.INVALID_ARGUMENT
    assert _add(gx, cache, None) == _evict(gx, cache, None) == gx.INVALID_ARGUMENT
    for field in ("weight", "position", "dropped"):
        broken = gx.KvWeights(weights.weight, weights.position, weights.dropped)
        setattr(broken, field, None)
        assert _add(gx, cache, broken) == _evict(gx, cache, broken) == gx.INVALID_ARGUMENT
        assert gx.lib().gfxinfer_launch_kv_weights_begin(_ref(cache), _ref(broken), _ids(0), _ids(1), 1, None) == gx.INVALID_ARGUMENT
    for tokens in (None, _ids(0), _ids((1 << 20) + 1)):
        assert gx.lib().gfxinfer_launch_kv_weights_begin(_ref(cache), _ref(weights), _ids(0), tokens, 1, None) == gx.INVALID_ARGUMENT


def test_workspace_sizes(gx, cache):  # noqa: F811
    assert gx.kv_pages_chunk_attention_workspace_bytes(cache, [1, 0, 2], 4) == 0      # a short table: positions are not divided
    assert gx.kv_weights_workspace_bytes(cache, [1, 0, 2], 4) > 0
    assert gx.kv_pages_evict_workspace_bytes(cache, 2, 20) > 0
    assert gx.kv_pages_evict_workspace_bytes(cache, 2, 1 << 30) > 0                   # no sequence reaches it
    for bad in (([], 4), ([0], 4), ([1], 3), ([1] * 257, 4), ([1 << 20, 1], 4)):
        assert gx.kv_pages_chunk_attention_workspace_bytes(cache, *bad) == 0
        assert gx.kv_weights_workspace_bytes(cache, *bad) == 0
    for bad in ((0, 20), (513, 20), (1, 0)):
        assert gx.kv_pages_evict_workspace_bytes(cache, *bad) == 0
    cache.table_stride = 1024
    assert gx.kv_pages_chunk_attention_workspace_bytes(cache, [1, 0, 2], 4) > 0
    assert _attention(gx, cache, bytes=gx.kv_pages_chunk_attention_workspace_bytes(cache, [1, 2], 4) - 1) == gx.INVALID_ARGUMENT
    assert "workspace" in gx.last_error()


def test_lists_of_the_wrappers(gx, cache, weights):  # noqa: F811
    for call in (lambda: gx.launch_kv_pages_chunk_attention(cache, 0, 0, None, 0, None, [0, 1], [1], 4, None),
                 lambda: gx.launch_kv_weights_begin(cache, weights, [0], [1, 1]),
                 lambda: gx.launch_kv_weights_add(cache, weights, 0, 0, 0, [0], [], 4, None)):
        with pytest.raises(ValueError):
            call()
