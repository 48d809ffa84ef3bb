"""CPU tests of the paged K/V cache's launchers: what they refuse, before anything is launched."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

LIMITS = dict(layers=2, page_count=8, page_tokens=16, kv_heads=2, head_size=128, sequences=4, table_stride=3)


def _aligned(size):
    raw = np.zeros(size + 16, dtype=np.uint8)
    return raw[(-raw.ctypes.data) % 16:][:size]


@pytest.fixture()
def cache(gx):
    """A description over host memory: enough for calls that are refused."""
    n = 2 * 8 * 16 * 2 * 128 * 2
    arrays = [_aligned(n), _aligned(n), _aligned(4 * 3 * 4), _aligned(4 * 4), _aligned(8 * 4)]
    pages = gx.KvPages(*(a.ctypes.data for a in arrays), *LIMITS.values())
    pages.tensors = arrays
    return pages


def _refused(gx, status, *words):
    assert status == gx.INVALID_ARGUMENT
    assert all(w in gx.last_error() for w in words), gx.last_error()


def _ids(*values):
    return (ctypes.c_uint32 * len(values))(*values)


def _calls(gx, pages, ids, count):
    """Every call that takes a list of sequences, with arguments that are otherwise good."""
    L, at = gx.lib(), ctypes.byref(pages) if pages is not None else None
    work = _aligned(1 << 16)
    rows = _aligned(4 * 4 * 512 * 4)
    status = _aligned(16)
    return {
        "fork": lambda: L.gfxinfer_launch_kv_pages_fork(at, 3, ids, count, None),
        "reserve": lambda: L.gfxinfer_launch_kv_pages_reserve(at, ids, count, 1, status.ctypes.data, work.ctypes.data,
                                                              work.nbytes, None),
        "append": lambda: L.gfxinfer_launch_kv_pages_append(at, 0, rows.ctypes.data, rows.ctypes.data, ids, count, 1, None),
        "advance": lambda: L.gfxinfer_launch_kv_pages_advance(at, ids, count, 1, None, None),
        "free": lambda: L.gfxinfer_launch_kv_pages_free(at, ids, None, count, None),
    }


@pytest.mark.parametrize("field,value", [
    ("key_pages", None), ("value_pages", None), ("page_table", None), ("lengths", None), ("references", None),
    ("layers", 0), ("page_count", 0), ("page_count", (1 << 24) + 1), ("page_tokens", 8), ("page_tokens", 24),
    ("page_tokens", 8192), ("kv_heads", 0), ("kv_heads", 1025), ("head_size", 64), ("head_size", 192),
    ("sequences", 0), ("sequences", 65537), ("table_stride", 0), ("table_stride", 1 << 28)])
def test_bad_descriptions_are_refused(gx, cache, field, value):
    setattr(cache, field, value)
    assert gx.kv_pages_workspace_bytes(cache) == 0
    for name, call in _calls(gx, cache, _ids(0), 1).items():
        _refused(gx, call(), "K/V page")
    _refused(gx, gx.lib().gfxinfer_launch_kv_pages_reset(ctypes.byref(cache), None), "K/V page")


def test_null_and_misaligned_descriptions_are_refused(gx, cache):
    for call in _calls(gx, None, _ids(0), 1).values():
        _refused(gx, call(), "null")
    for field in ("key_pages", "value_pages", "references"):
        whole = getattr(cache, field)
        setattr(cache, field, whole + 4)
        _refused(gx, gx.lib().gfxinfer_launch_kv_pages_reset(ctypes.byref(cache), None), "aligned")
        setattr(cache, field, whole)


@pytest.mark.parametrize("ids,count", [((), 0), ((0,), 0), (tuple(range(4)) * 200, 513), ((4,), 1), ((0, 0), 2), ((1, 2, 1), 3)])
def test_bad_lists_are_refused(gx, cache, ids, count):
    for name, call in _calls(gx, cache, _ids(*ids), count).items():
        _refused(gx, call())


def test_default_list_must_fit_the_cache(gx, cache):
    for name, call in _calls(gx, cache, None, 5).items():
        _refused(gx, call())


def test_call_arguments_are_checked(gx, cache):
    L, at = gx.lib(), ctypes.byref(cache)
    work, status, rows = _aligned(1 << 16), _aligned(16), _aligned(1 << 16)
    w, st, r = work.ctypes.data, status.ctypes.data, rows.ctypes.data
    need = gx.kv_pages_workspace_bytes(cache)
    assert 0 < need <= work.nbytes
    _refused(gx, L.gfxinfer_launch_kv_pages_fork(at, 4, _ids(0), 1, None), "parent")
    _refused(gx, L.gfxinfer_launch_kv_pages_fork(at, 0, None, 1, None), "children")
    _refused(gx, L.gfxinfer_launch_kv_pages_fork(at, 1, _ids(0, 1), 2, None), "onto itself")
    for tokens, s, ws, size, word in ((0, st, w, need, "tokens"), ((1 << 24) + 1, st, w, need, "tokens"),
                                      (1, None, w, need, "status"), (1, st, None, need, "workspace"),
                                      (1, st, w + 8, need, "workspace"), (1, st, w, need - 1, "workspace")):
        _refused(gx, L.gfxinfer_launch_kv_pages_reserve(at, _ids(0), 1, tokens, s, ws, size, None), word)
    for layer, k, v, tokens in ((2, r, r, 1), (0, None, r, 1), (0, r, None, 1), (0, r + 2, r, 1), (0, r, r + 4, 1), (0, r, r, 0)):
        _refused(gx, L.gfxinfer_launch_kv_pages_append(at, layer, k, v, _ids(0), 1, tokens, None), "append")
    _refused(gx, L.gfxinfer_launch_kv_pages_append(at, 0, r, r, _ids(0), 1, (1 << 31) // 32 + 1, None), "too many")
    _refused(gx, L.gfxinfer_launch_kv_pages_compact(at, None, w, need - 1, None), "workspace")
    for a, b, n in (((0,), (0,), 1), ((0, 1), (2, 2), 2), ((0, 1), (1, 2), 2), ((8,), (0,), 1), ((0,), (8,), 1), ((0,), (1,), 0),
                    (tuple(range(8)) * 40, tuple(range(8)) * 40, 257)):
        _refused(gx, L.gfxinfer_launch_kv_pages_copy(at, _ids(*a), _ids(*b), n, None))
    _refused(gx, L.gfxinfer_launch_kv_pages_copy(at, None, _ids(1), 1, None))
    _refused(gx, L.gfxinfer_launch_kv_pages_copy(at, _ids(1), None, 1, None))


def test_descriptions_from_tensors_check_shapes(gx):
    import torch
    k = torch.zeros(2, 8, 16, 2, 128, dtype=torch.float16)
    table, lengths, references = (torch.zeros(s, dtype=torch.int32) for s in ((4, 3), (4,), (8,)))
    pages = gx.KvPages.of(k, torch.zeros_like(k), table, lengths, references)
    assert {n: getattr(pages, n) for n in LIMITS} == LIMITS
    for bad in ((k, k[:1], table, lengths, references), (k, k, table, lengths[:3], references),
                (k, k, table, lengths, references[:7]), (k.float(), k, table, lengths, references),
                (k, k.transpose(1, 2).contiguous().transpose(1, 2), table, lengths, references),
                (k, k, table.long(), lengths, references)):
        with pytest.raises(ValueError):
            gx.KvPages.of(*bad)


def test_pages_are_not_bfloat16_and_lists_are_whole_numbers(gx):
    import array

    import torch
    pool = torch.zeros((1, 4, 16, 2, 128), dtype=torch.bfloat16)
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError):
        gx.KvPages.of(pool, pool, i(3, 4), i(3), i(4))
    pages = gx.KvPages.of(pool.half(), pool.half(), i(3, 4), i(3), i(4))
    for bad in (array.array("f", [1.0]), [1.5]):
        with pytest.raises(TypeError):
            gx.launch_kv_pages_fork(pages, 0, bad, stream=0)
    with pytest.raises(OverflowError):
        gx.launch_kv_pages_fork(pages, 0, [-1], stream=0)
    with pytest.raises(gx.GfxinferError):
        gx.launch_kv_pages_fork(pages, 0, array.array("I", [9]), stream=0)
