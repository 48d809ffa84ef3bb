"""CPU tests of the wrappers of weights and eviction: weights that were made for other pages are refused before a call."""
from __future__ import annotations

import pytest
import torch


def _pages(gx, sequences, columns, page_tokens=16):
    pool = torch.zeros(1, 4, page_tokens, 1, 128, dtype=torch.float16)
    return gx.KvPages.of(pool, torch.zeros_like(pool), torch.zeros(sequences, columns, dtype=torch.int32),
                         torch.zeros(sequences, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))


def _weights(gx, pages):
    rows = (pages.sequences, pages.table_stride * pages.page_tokens)
    return gx.KvWeights.of(pages, torch.zeros(rows), torch.zeros(rows, dtype=torch.int32), torch.zeros(rows[0], dtype=torch.int32))


def _calls(gx, pages, weights):
    return (lambda: gx.launch_kv_weights_begin(pages, weights, [0], [1]),
            lambda: gx.launch_kv_weights_add(pages, weights, 0, 0, 0, [0], [1], 1, None),
            lambda: gx.launch_kv_pages_evict(pages, weights, [0], 4, 0, 0, 0, None))


@pytest.mark.parametrize("sequences,columns,page_tokens", [(3, 2, 16), (2, 3, 16), (2, 2, 32), (2, 1, 16), (1, 2, 16)])
def test_weights_of_other_pages_are_refused(gx, monkeypatch, sequences, columns, page_tokens):
    """A table with more columns or sequences would let the call write behind the weights' tensors."""
    weights = _weights(gx, _pages(gx, 2, 2))
    called = []
    for name in ("gfxinfer_launch_kv_weights_begin", "gfxinfer_launch_kv_weights_add", "gfxinfer_launch_kv_pages_evict"):
        monkeypatch.setattr(gx.lib(), name, lambda *a, name=name: called.append(name) or 1)
    for call in _calls(gx, _pages(gx, sequences, columns, page_tokens), weights):
        with pytest.raises(ValueError, match="K/V weights"):
            call()
    assert not called


def test_weights_of_another_device_are_refused(gx, monkeypatch):
    pages = _pages(gx, 2, 2)
    weights = _weights(gx, pages)
    pages.device = 0
    for name in ("gfxinfer_launch_kv_weights_begin", "gfxinfer_launch_kv_weights_add", "gfxinfer_launch_kv_pages_evict"):
        monkeypatch.setattr(gx.lib(), name, lambda *a: 1)
    for call in _calls(gx, pages, weights):
        with pytest.raises(ValueError, match="another device"):
            call()


def test_weights_of_the_same_shape_and_plain_addresses_pass(gx, monkeypatch):
    """Pages described anew, and weights that are addresses, which are the caller's to know."""
    pages = _pages(gx, 2, 2)
    weights = _weights(gx, pages)
    again = _pages(gx, 2, 2)
    for x in (pages, again):
        x.device = weights.device = None
    bare = gx.KvWeights(weights.weight, weights.position, weights.dropped)
    called = []
    monkeypatch.setattr(gx.lib(), "gfxinfer_launch_kv_weights_begin", lambda *a: called.append(a) or 0)
    monkeypatch.setattr(gx, "_launch_stream", lambda device, stream: None)
    for w in (weights, bare):
        gx.launch_kv_weights_begin(again, w, [0], [1])
    assert len(called) == 2
