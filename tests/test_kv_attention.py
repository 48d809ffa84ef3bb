"""CPU tests of the paged attention launcher: what it refuses, before anything is launched."""
from __future__ import annotations

import ctypes

import pytest

from test_kv_pages import _aligned, _ids, cache  # noqa: F401  (the fixture)


def _call(gx, pages, **change):
    a = dict(layer=0, query=_aligned(4096), gate=_aligned(4096), output=_aligned(4096), ids=_ids(0, 1), count=2, tokens=1,
             q_heads=4, shared=0, workspace=_aligned(1 << 20), bytes=1 << 20)
    a.update(change)
    at = lambda x: x if x is None or isinstance(x, int) else x.ctypes.data  # noqa: E731
    return gx.lib().gfxinfer_launch_kv_pages_gated_attention(
        None if pages is None else ctypes.byref(pages), a["layer"], at(a["query"]), at(a["gate"]), at(a["output"]), a["ids"],
        a["count"], a["tokens"], a["q_heads"], a["shared"], at(a["workspace"]), a["bytes"], None)


@pytest.mark.parametrize("change", [
    dict(layer=2), dict(query=None), dict(output=None), dict(count=0), dict(count=513), dict(tokens=0), dict(tokens=33),
    dict(q_heads=0), dict(q_heads=3), dict(q_heads=1026), dict(shared=49), dict(workspace=None), dict(bytes=100),
    dict(ids=_ids(0, 4)), dict(ids=None, count=5), dict(query=_aligned(4096).ctypes.data + 2),
    dict(output=_aligned(4096).ctypes.data + 2), dict(gate=_aligned(4096).ctypes.data + 4),
    dict(workspace=_aligned(1 << 20).ctypes.data + 8)])
def test_bad_arguments_are_refused(gx, cache, change):  # noqa: F811
    assert _call(gx, cache, **change) == gx.INVALID_ARGUMENT
    assert gx.last_error()


def test_null_pages_and_bad_workspace_sizes(gx, cache):  # noqa: F811
    assert _call(gx, None) == gx.INVALID_ARGUMENT
    for bad in ((0, 1, 4, 0), (1, 0, 4, 0), (1, 33, 4, 0), (1, 1, 3, 0), (1, 1, 4, 49), (513, 1, 4, 0)):
        assert gx.kv_pages_attention_workspace_bytes(cache, *bad) == 0
    need = gx.kv_pages_attention_workspace_bytes(cache, 2, 1, 4, 16)
    assert need > 0
    assert _call(gx, cache, shared=16, bytes=need - 1) == gx.INVALID_ARGUMENT
    assert "workspace" in gx.last_error()
