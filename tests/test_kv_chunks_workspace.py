"""The workspace of chunk attention: what is divided needs it, however many tokens there are besides."""
from __future__ import annotations

import numpy as np
import pytest

from test_kv_pages import cache  # noqa: F401  (the fixture)

MOST = 104 << 20  # 2 x 256 + 255 workgroups' rows at head size 256: (767 * 128) * (256 + 2) * 4 bytes


@pytest.mark.parametrize("heads", [(40, 8, 128), (24, 4, 256), (64, 8, 128), (32, 1, 256), (16, 16, 128)])
def test_the_size_is_bounded(gx, cache, heads):  # noqa: F811
    """Parts of all rows were counted where only the last tiles are divided: gigabytes for 16 tiles of 10256."""
    q_heads, cache.kv_heads, cache.head_size = heads
    cache.page_tokens, cache.table_stride, cache.sequences = 64, 1024, 256
    rng = np.random.default_rng(q_heads)
    some = 0
    for tokens in [[n] for n in (1, 8, 300, 2048, 8192, 8200, 32768, 32800, 100000, (1 << 20) - 1)] + [
            [1] * n for n in (1, 8, 31, 64, 65, 100, 200, 256)] + [rng.integers(0, 4000, int(n)).tolist() + [1] for n in rng.integers(1, 200, 60)]:
        size = gx.kv_pages_chunk_attention_workspace_bytes(cache, tokens, q_heads)
        assert 0 <= size <= MOST, (tokens[:5], len(tokens), size)
        some += size > 0
    assert some > 10


@pytest.mark.gpu
@pytest.mark.parametrize("heads,page,lengths,tokens", [
    ((32, 1, 256), 32, [100, 60], [1050, 1]),                 # 263 items of 256 rows, 7 divided
    ((32, 1, 128), 64, [300, 5, 700, 33], [2070, 2, 0, 1]),   # 518 + 2
    ((8, 2, 128), 16, [700, 64, 1200, 3], [4100, 1, 4150, 40]),  # the rest lies in two sequences
    ((6, 6, 128), 16, [900] * 90, [1] * 90),                  # decoding sequences alone: 540 items
    ((12, 4, 256), 16, [900, 30] * 40, [1, 3] * 40),
])
def test_parts_of_the_rest_stay_in_the_workspace(device, gx, heads, page, lengths, tokens):
    import torch

    from gpu_util import dev, host, say
    from test_kv_chunks_gpu import Chunks
    say("parts of the rest", heads, page, lengths[:4], tokens[:4])
    c = Chunks(np.random.default_rng(sum(tokens)), heads, page, lengths, tokens, gap=40)
    pages, rows = c.pages(gx), sum(tokens)
    size = gx.kv_pages_chunk_attention_workspace_bytes(pages, tokens, heads[0])
    work = torch.full((size + 4096,), 0xff, dtype=torch.uint8, device="cuda")
    out = torch.full((rows, heads[0], heads[2]), 7.0, dtype=torch.float16, device="cuda")
    sums = torch.full((rows, heads[0]), 7.0, device="cuda")
    for _ in range(2):                                        # the second time with what the first one left there
        gx.launch_kv_pages_chunk_attention(pages, 1, dev(c.query), dev(c.gate), out, sums, range(len(tokens)), tokens, heads[0], work[:size])
        which = [i for i in range(len(tokens)) if tokens[i]]
        c.check(host(out), host(sums), which if len(which) < 10 else which[::9] + which[-1:])
        assert bool((work[size:] == 0xff).all())


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(40, 8, 128), (24, 4, 256)])
def test_sequences_without_tokens_change_nothing(device, gx, heads):
    """A long one listed with no new tokens: the others are divided as without it, so their results have the same bits."""
    from gpu_util import say
    from test_kv_chunks_gpu import Chunks
    say("idle sequences", heads)
    c = Chunks(np.random.default_rng(6), heads, 64, [600, 1100, 9000, 200], [1, 3, 0, 1])
    with_it = c.run(gx)
    c.check(*with_it, [0, 1, 3])
    c.tokens = [1, 3, 1]
    without = c.run(gx, listed=[0, 1, 3])
    for a, b in zip(with_it, without):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("heads,count", [((40, 8, 128), 64), ((40, 8, 128), 95), ((24, 4, 256), 64), ((24, 4, 256), 100)])
def test_decoding_sequences_are_divided(gx, cache, heads, count):  # noqa: F811
    """One more workgroup a place is worth it where lengths differ: a long sequence among 64 was a single range."""
    q_heads, cache.kv_heads, cache.head_size = heads
    cache.page_tokens, cache.table_stride, cache.sequences = 64, 1024, 256
    size = gx.kv_pages_chunk_attention_workspace_bytes(cache, [1] * count, q_heads)
    assert size >= 2 * count * q_heads * (heads[2] + 2) * 4
