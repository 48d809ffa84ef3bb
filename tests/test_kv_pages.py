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


def _tensor_calls(gx, pages, **change):
    """Every wrapper that takes tensors beside the description: addresses (not looked at) but for what `change` gives."""
    a = dict.fromkeys(("key", "value", "status", "token_counts", "live", "query", "gate", "output"), 4096)
    a.update(work=None)
    a.update(change)
    return {
        "append": lambda: gx.launch_kv_pages_append(pages, 0, a["key"], a["value"], [0, 1], 3, stream=0),
        "reserve": lambda: gx.launch_kv_pages_reserve(pages, [0, 1], 3, a["status"], a["work"], stream=0),
        "advance": lambda: gx.launch_kv_pages_advance(pages, [0, 1], 3, a["token_counts"], stream=0),
        "compact": lambda: gx.launch_kv_pages_compact(pages, a["live"], a["work"], stream=0),
        "attention": lambda: gx.launch_kv_pages_gated_attention(pages, 0, a["query"], a["gate"], a["output"], [0, 1], 3, 4, 0,
                                                                a["work"], stream=0),
    }


@pytest.fixture()
def tensor_pages(gx):
    import torch
    k = torch.zeros(2, 8, 16, 2, 128, dtype=torch.float16)
    return gx.KvPages.of(k, k, *(torch.zeros(s, dtype=torch.int32) for s in ((4, 3), (4,), (8,))))


def _bad_tensors():
    import torch
    z = torch.zeros
    h, w = torch.float16, torch.int32
    return [
        ("append", dict(key=z(2, 3, 256)), "key"), ("append", dict(key=z(2, 3, 256, dtype=torch.bfloat16)), "key"),
        ("append", dict(key=z(2, 3, 255, dtype=h)), "key"), ("append", dict(key=z(256, 3, 2, dtype=h).permute(2, 1, 0)), "key"),
        ("append", dict(key=np.zeros((2, 3, 256), np.float16)), "key"), ("append", dict(value=z(2, 3, 256, dtype=h)), "value"),
        ("append", dict(value=z(2, 2, 256)), "value"), ("append", dict(value=z(2, 3, 256).double()), "value"),
        ("reserve", dict(status=z(1, dtype=torch.int64)), "status"), ("reserve", dict(status=z(0, dtype=w)), "status"),
        ("reserve", dict(work=z(4096, 2, dtype=w)[:, 0]), "workspace"),
        ("advance", dict(token_counts=z(2, dtype=torch.int64)), "token_counts"), ("advance", dict(token_counts=z(2)), "token_counts"),
        ("advance", dict(token_counts=z(1, dtype=w)), "token_counts"), ("advance", dict(token_counts=z(4, dtype=w)[::2]), "token_counts"),
        ("compact", dict(live=z(1)), "live_pages"), ("compact", dict(live=z(0, dtype=w)), "live_pages"),
        ("attention", dict(query=z(2, 3, 4, 128)), "query"), ("attention", dict(query=z(2, 2, 4, 128, dtype=h)), "query"),
        ("attention", dict(query=z(2, 4, 3, 128, dtype=h).transpose(1, 2)), "query"),
        ("attention", dict(gate=z(2, 3, 4, 256, dtype=h)), "gate"), ("attention", dict(gate=z(2, 3, 4, 128)), "gate"),
        ("attention", dict(output=z(2, 3, 4, 128)), "output"), ("attention", dict(output=z(2, 3, 3, 128, dtype=h)), "output"),
        ("attention", dict(work=z(1, dtype=w).expand(4096)), "workspace"),
    ]


@pytest.mark.parametrize("at", range(25))
def test_operands_of_other_types_or_sizes_are_refused(gx, tensor_pages, at):
    """Before the library is called: what a kernel would read or write past the end of, or take for other numbers."""
    name, change, word = _bad_tensors()[at]
    tensor_pages.device = None                                # of no device, as a description from addresses
    with pytest.raises(ValueError, match=word):
        _tensor_calls(gx, tensor_pages, **change)[name]()


def test_host_memory_is_refused(gx, tensor_pages):
    """Good tensors that no GPU reaches, and a cache in such memory."""
    import torch
    assert len(_bad_tensors()) == 25
    assert tensor_pages.device == -1
    tensor_pages.device = None
    z, h, w = torch.zeros, torch.float16, torch.int32
    for name, change in (("append", dict(key=z(2, 3, 256, dtype=h))), ("append", dict(value=z(2, 3, 256))),
                         ("reserve", dict(status=z(1, dtype=w))), ("reserve", dict(work=z(4096, dtype=w))),
                         ("advance", dict(token_counts=z(2, dtype=w))), ("compact", dict(live=z(1, dtype=w))),
                         ("compact", dict(work=z(4096))), ("attention", dict(query=z(2, 3, 4, 128, dtype=h))),
                         ("attention", dict(gate=z(2, 3, 4, 256))), ("attention", dict(output=z(2, 3, 4, 128, dtype=h))),
                         ("attention", dict(work=z(4096)))):
        with pytest.raises(ValueError, match="memory"):
            _tensor_calls(gx, tensor_pages, **change)[name]()
    tensor_pages.device = -1
    calls = [lambda: gx.launch_kv_pages_reset(tensor_pages, stream=0), lambda: gx.launch_kv_pages_fork(tensor_pages, 0, [1], stream=0),
             lambda: gx.launch_kv_pages_free(tensor_pages, [1], stream=0), lambda: gx.launch_kv_pages_copy(tensor_pages, [1], [2], stream=0)]
    for call in calls + list(_tensor_calls(gx, tensor_pages).values()):
        with pytest.raises(gx.GfxinferError, match="memory"):
            call()
    pools = tensor_pages.tensors
    with pytest.raises(ValueError):
        gx.KvPages.of(pools[0], pools[1], torch.zeros(4, 3), pools[3], pools[4])
