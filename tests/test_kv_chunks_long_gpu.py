"""Chunk attention over long caches: more ranges than a wave has lanes, more steps of a range than there are marks for strange values."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import dev, host, say
from test_kv_chunks_gpu import A, B, Chunks

pytestmark = pytest.mark.gpu


def _ranges(gx, c):
    """Ranges of a call whose tiles are all divided, by the size of its workspace."""
    q_heads, _, d = c.heads
    size = gx.kv_pages_chunk_attention_workspace_bytes(c.pages(gx), c.tokens, q_heads)
    return size // (sum(c.tokens) * q_heads * (d + 2) * 4)


@pytest.mark.parametrize("heads,length", [(A, 12000), (B, 9000)])
@pytest.mark.parametrize("tokens", [1, 3, 8])
@pytest.mark.parametrize("highest", [0.02, 0.99, None])
def test_more_ranges_than_lanes(device, gx, heads, length, tokens, highest):
    """The largest scores in the first ranges, in the last ones, or anywhere: the join goes on from the ranges before."""
    q_heads, kv_heads, d = heads
    c = Chunks(np.random.default_rng(tokens), heads, 64, [length], [tokens])
    if highest is not None:
        c.query[..., 0] = 4
        k = c.rows[0][0]
        k[:, :, 0] = -1
        k[int(length * highest):int(length * highest) + 5, :, 0] = 6 * d ** 0.5 / 4  # 6 to 9 nats above the others
        for j in range(len(k)):
            c.put(0, j, k=k[j])
    if tokens * q_heads // kv_heads <= 32:
        assert _ranges(gx, c) > 64
    say("more ranges than lanes", heads, length, tokens, highest, _ranges(gx, c))
    got, sums = c.run(gx)
    c.check(got, sums)


@pytest.mark.parametrize("heads,length", [(A, 12000), (B, 9000)])
def test_strange_values_in_a_late_range(device, gx, heads, length):
    q_heads, kv_heads, d = heads
    group = q_heads // kv_heads
    c = Chunks(np.random.default_rng(3), heads, 64, [length], [2])
    assert _ranges(gx, c) > 64
    good = {}
    for at, head, dim, value in ((length - 100, 0, 3, np.inf), (length - 3, 1, 5, -np.inf), (length - 500, 2, d - 1, np.nan)):
        good[at] = c.rows[0][1][at].copy()
        v = good[at].copy()
        v[head, dim] = value
        c.put(0, at, v=v)
    say("strange values in a late range", heads)
    got, sums = c.run(gx)
    got = got.copy()
    assert np.all(got[:, :group, 3] == np.inf) and np.all(got[:, group:2 * group, 5] == -np.inf)
    assert np.isnan(got[:, 2 * group:3 * group, d - 1]).all()
    for at, v in good.items():
        c.put(0, at, v=v)
    _fill(c, got, [(h, dim) for head, dim in ((0, 3), (1, 5), (2, d - 1)) for h in range(head * group, head * group + group)])
    c.check(got, sums)


def _fill(c, got, places):
    """Puts the definition where a test has looked already."""
    d = c.heads[2]
    for h, dim in places:
        s, _, v = c.rows_of(0, h)
        w = np.exp(s - s.max(1, keepdims=True))
        got[:, h, dim] = (w @ v[:, dim]) / w.sum(1) / (1 + np.exp(-c.gate[:, h, d + dim].astype(np.float64)))


@pytest.mark.parametrize("heads,length,listed", [((2, 2, 128), 66500, 256), ((4, 4, 256), 33500, 64)])
def test_more_steps_than_marks(device, gx, heads, length, listed):
    """A range of more than 1024 steps, strange values in steps 2 and 1026, whose marks are one, and in another: one sequence is
    listed so often that no tile is divided."""
    import torch
    q_heads, kv_heads, d = heads
    step, tokens = 8192 // d, 33
    c = Chunks(np.random.default_rng(d), heads, 256, [length], [tokens], gap=0)
    pages, many = c.pages(gx), [tokens] * listed
    assert gx.kv_pages_chunk_attention_workspace_bytes(pages, many, q_heads) == 0 and length > 1030 * step
    strange = [(2 * step + 7, 0, 3, np.inf), (1026 * step + 9, 1, 5, -np.inf), (700 * step, 0, d - 1, np.nan), (length + 20, 1, 8, np.nan)]
    good = [(at, c.rows[0][1][at].copy()) for at, *_ in strange]
    for at, head, dim, value in strange:
        v = c.rows[0][1][at].copy()
        v[head, dim] = value
        c.put(0, at, v=v)
    pages = c.pages(gx)
    query, gate = (torch.from_numpy(x).cuda().repeat(listed, 1, 1) for x in (c.query, c.gate))
    out = torch.zeros(tokens * listed, q_heads, d, dtype=torch.float16, device="cuda")
    sums = torch.zeros(tokens * listed, q_heads, device="cuda")
    say("more steps than marks", heads, length)
    gx.launch_kv_pages_chunk_attention(pages, 1, query, gate, out, sums, [0] * listed, many, q_heads, None)
    bits = out.view(torch.int16).view(listed, -1)
    assert bool((bits == bits[0]).all()) and bool((sums.view(listed, -1) == sums.view(listed, -1)[0]).all())
    got = host(out[:tokens]).copy()
    assert np.all(got[:, 0, 3] == np.inf) and np.all(got[:, 1, 5] == -np.inf) and np.isnan(got[:, 0, d - 1]).all()
    assert np.isnan(got[20:, 1, 8]).all() and not np.isnan(got[:20, 1, 8]).any()
    for at, v in good:
        c.put(0, at, v=v)
    _fill(c, got, [(0, 3), (1, 5), (0, d - 1)])
    got[20:, 1, 8], kept = 0, got[:20, 1, 8].copy()
    rest = got.copy()
    _fill(c, rest, [(1, 8)])
    rest[:20, 1, 8] = kept
    c.check(rest, host(sums[:tokens]))
