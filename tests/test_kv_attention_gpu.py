"""Paged attention with a shared prefix on the GPU against the definition in 64 bits.

Tolerance.  u = 2^-24 is half a step of fp32.  A score is a sum of D products accumulated in fp32: off by at most
D u |q|.|k| / sqrt(D), and scaling, the difference to the maximum and the exponential add a few u of the score and of the
weight.  A weight is therefore off by e = 2 (D + 8) u max(|q|.|k|) / sqrt(D) + 2^-21 relatively (twice: against the maximum
too; 2^-21 covers the exponential and the fp16 pair that carries a weight), numerator and denominator both.  A wave sums
at most a quarter of the positions, in at most two additions each, and the merges add a few dozen more: (n / 2 + 64) u.
The sum of both, times the weighted mean of |v| and the gate, is added to the half step of the fp16 result (2^-11
relatively, 2^-25 below the normal numbers).
"""
from __future__ import annotations

import math

import numpy as np
import pytest

from gpu_util import dev, host, say

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


class Problem:
    """Two layers of pages in no order; what no sequence sees is NaN: rows past the ends, free pages, layer 0."""

    def __init__(self, rng, q_heads, kv_heads, d, page, lengths, tokens, shared, gate=True, slack=3, spread=1.0):
        self.heads, self.page, self.lengths, self.tokens, self.shared = (q_heads, kv_heads, d), page, lengths, tokens, shared
        n = len(lengths)
        held = [-(-(x + tokens) // page) for x in lengths]
        common = shared // page
        pages = common + sum(h - common for h in held) + slack
        order = rng.permutation(pages).tolist()
        self.k, self.v = (np.full((2, pages, page, kv_heads, d), np.nan, np.float16) for _ in range(2))
        self.table = np.full((n + 1, max(held) + 1), -1, np.int32)
        self.references = np.zeros(pages, np.int32)
        prefix = [rng.standard_normal((shared, kv_heads, d)).astype(np.float16) * spread for _ in range(2)]
        self.rows = []
        at = common
        for i, h in enumerate(held):
            mine = order[:common] + order[at:at + h - common]
            at += h - common
            self.table[i, :h] = mine
            self.references[mine] += 1
            own = [rng.standard_normal((lengths[i] + tokens - shared, kv_heads, d)).astype(np.float16) * spread for _ in range(2)]
            kv = [np.concatenate([a, b]).astype(np.float16) for a, b in zip(prefix, own)]
            self.rows.append(kv)
            for pool, x in zip((self.k, self.v), kv):
                for j in range(0, len(x), page):
                    pool[1, mine[j // page], :len(x[j:j + page])] = x[j:j + page]
        self.query = rng.standard_normal((n, tokens, q_heads, d)).astype(np.float16)
        self.gate = (rng.standard_normal((n, tokens, q_heads, 2 * d)) * 2).astype(np.float32) if gate else None
        if gate:
            self.gate[..., :d] = np.nan                       # the query half of the projection is not read

    def put(self, i, position, k=None, v=None):
        """Overwrites rows of one position of one sequence, in its page and in the reference."""
        for pool, rows, x in ((self.k, self.rows[i][0], k), (self.v, self.rows[i][1], v)):
            if x is not None:
                rows[position] = x
                pool[1, self.table[i, position // self.page], position % self.page] = x

    def run(self, gx, listed=None, shared=None, stream=None):
        import torch
        q_heads, kv_heads, d = self.heads
        listed = list(range(len(self.lengths))) if listed is None else listed
        shared = self.shared if shared is None else shared
        keep = [dev(x) for x in (self.k, self.v, self.table, np.array(self.lengths + [0], np.int32), self.references)]
        pages = gx.KvPages.of(*keep)
        query = dev(self.query[listed])
        gate = dev(self.gate[listed]) if self.gate is not None else None
        out = torch.full((len(listed) + 1, self.tokens, q_heads, d), 7.0, dtype=torch.float16, device="cuda")
        work = torch.full((gx.kv_pages_attention_workspace_bytes(pages, len(listed), self.tokens, q_heads, shared),), 0xff,
                          dtype=torch.uint8, device="cuda")
        gx.launch_kv_pages_gated_attention(pages, 1, query, gate, out, listed, self.tokens, q_heads, shared, work, stream=stream)
        got = host(out)
        assert np.all(got[-1] == 7.0)                         # rows behind the last sequence stay
        return got[:-1]

    def expect(self, i):
        """(result, tolerance) of sequence i, [tokens, q_heads, d]."""
        q_heads, kv_heads, d = self.heads
        group = q_heads // kv_heads
        k, v = (x.astype(np.float64) for x in self.rows[i])
        want, tol = np.zeros((self.tokens, q_heads, d)), np.zeros((self.tokens, q_heads, d))
        for t in range(self.tokens):
            n = self.lengths[i] + t + 1
            for h in range(q_heads):
                q, kk, vv = self.query[i, t, h].astype(np.float64), k[:n, h // group], v[:n, h // group]
                s = kk @ q / math.sqrt(d)
                w = np.exp(s - s.max())
                w /= w.sum()
                e = 2 * (d + 8) * U * (np.abs(kk) @ np.abs(q)).max() / math.sqrt(d) + 2.0 ** -21
                g = 1 / (1 + np.exp(-self.gate[i, t, h, d:].astype(np.float64))) if self.gate is not None else 1.0
                want[t, h] = w @ vv * g
                tol[t, h] = (2 * e + (n / 2 + 64) * U) * (w @ np.abs(vv)) * g
        return want, tol + np.maximum(np.abs(want) * 2.0 ** -11, 2.0 ** -25) * (1 + 2.0 ** -10)

    def check(self, got, listed=None):
        for at, i in enumerate(range(len(self.lengths)) if listed is None else listed):
            want, tol = self.expect(i)
            assert np.all(np.abs(got[at].astype(np.float64) - want) <= tol), (i, float(np.max(np.abs(got[at] - want) / tol)))


A, B = (40, 8, 128), (24, 4, 256)


@pytest.mark.parametrize("heads,page,lengths,tokens,shared", [
    ((1, 1, 128), 16, [0], 1, 0),                             # one position: the token itself
    ((1, 1, 256), 16, [0, 1, 2], 1, 0),
    ((2, 1, 128), 16, [0, 15, 16, 17, 31, 32, 33], 1, 0),
    ((6, 2, 128), 32, [16, 16, 40], 1, 16),                   # the prefix is all that some have
    ((16, 1, 128), 16, [100, 130], 1, 96),                    # 16 rows a sequence: full tiles
    ((17, 1, 128), 64, [100, 130], 1, 65),                    # 17: one row in the second tile
    (A, 16, [509, 512, 530, 600], 1, 509),
    (A, 64, [700] * 3 + [1500, 701], 5, 700),
    (A, 128, [300, 290, 333], 32, 289),                       # a full block of 32 tokens, two tiles of rows and more
    (A, 16, [77], 9, 0),
    (A, 256, [2100] * 14, 1, 2048),
    (B, 16, [509, 512, 530, 600], 1, 500),
    (B, 32, [200, 300, 201], 5, 200),
    (B, 64, [129, 257], 32, 100),
    (B, 4096, [5000, 4990], 2, 4987),                         # pages longer than a split
    ((8, 8, 128), 16, list(range(40, 73)), 1, 40),            # no grouping, 33 sequences
    ((24, 3, 256), 16, list(range(1, 20)), 3, 0),
])
@pytest.mark.parametrize("gate", [True, False])
def test_attention_equals_the_definition(device, gx, heads, page, lengths, tokens, shared, gate):
    rng = np.random.default_rng(len(lengths) * 1000 + page + shared)
    p = Problem(rng, *heads, page, lengths, tokens, shared, gate)
    say("paged attention", heads, page, lengths[:6], tokens, shared, gate)
    p.check(p.run(gx))


@pytest.mark.parametrize("heads", [A, B])
def test_prefix_length_only_changes_the_order_of_sums(device, gx, heads):
    rng = np.random.default_rng(3)
    p = Problem(rng, *heads, 32, [400, 431, 500], 2, 400)
    say("prefix lengths", heads)
    for shared in (0, 1, 31, 200, 399, 400):
        p.check(p.run(gx, shared=shared))


def test_listed_sequences_in_any_order_and_twice(device, gx):
    rng = np.random.default_rng(4)
    p = Problem(rng, *A, 16, [64, 80, 70, 99], 1, 64)
    say("listed sequences")
    for listed in ([3, 0], [2, 2, 1], [1]):
        p.check(p.run(gx, listed=listed), listed)


def test_large_scores_and_late_maxima(device, gx):
    """Scores of some hundreds, growing along the context: the running maximum moves in every block."""
    rng = np.random.default_rng(5)
    p = Problem(rng, *A, 16, [300, 310], 1, 256, spread=4.0)
    for i in range(2):
        for at in range(256, p.lengths[i] + 1):
            p.put(i, at, k=(p.rows[i][0][at] * np.float16(1 + (at - 256) / 32)))
    say("large scores")
    p.check(p.run(gx))


def test_strange_values_stay_where_they_are_seen(device, gx):
    """Infinities and NaN in positions of later tokens of a block do not reach earlier ones; visible ones do."""
    rng = np.random.default_rng(6)
    for heads in (A, B):
        p = Problem(rng, *heads, 16, [40, 75], 4, 32)
        kv_heads, d = heads[1], heads[2]
        p.check(p.run(gx))
        bad = rng.standard_normal((kv_heads, d)).astype(np.float16)
        bad[0, 3], bad[1, 5], bad[2, 0] = np.inf, np.nan, -np.inf
        p.put(0, 42, v=bad)                                   # token 2 of sequence 0 sees it first
        p.put(1, 78, k=np.full((kv_heads, d), np.nan, np.float16))   # token 3 of sequence 1
        say("strange values", heads)
        got = p.run(gx)
        group = heads[0] // kv_heads
        touched = np.zeros(got.shape, bool)
        for head, dim in ((0, 3), (1, 5), (2, 0)):
            touched[0, 2:, head * group:(head + 1) * group, dim] = True
        touched[1, 3] = True
        assert np.array_equal(np.isfinite(got), ~touched)
        assert np.all(got[0, 2:, :group, 3] == np.inf) and np.all(got[0, 2:, 2 * group:3 * group, 0] == -np.inf)
        # The rows that do not see them: the block's products are added one by one there and by 32s otherwise, two orders
        # of the same sum, each within the tolerance of the definition.
        p.rows = [[np.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0) for x in rows] for rows in p.rows]
        for i, first in ((0, 2), (1, 3)):
            want, tol = p.expect(i)
            assert np.all(np.abs(got[i, :first].astype(np.float64) - want[:first]) <= tol[:first])


def test_nan_queries_give_nan_and_missing_pages_zeros(device, gx):
    rng = np.random.default_rng(7)
    p = Problem(rng, *A, 16, [40, 50], 1, 0)
    p.query[0, 0, 7] = np.nan
    say("nan query")
    got = p.run(gx)
    assert np.all(np.isnan(got[0, 0, 7])) and np.isfinite(np.delete(got[0, 0], 7, 0)).all() and np.isfinite(got[1]).all()
    p.query[0, 0, 7] = 0
    p.table[0] = -1                                           # no page at all: nothing is seen
    p.table[1, 2] = 10000                                     # one page outside the pool: its positions are not seen
    got = p.run(gx)
    assert np.all(got[0] == 0)
    p.rows[1] = [np.concatenate([x[:32], x[48:]]) for x in p.rows[1]]
    p.lengths = [40, 34]
    want, tol = p.expect(1)
    assert np.all(np.abs(got[1] - want) <= tol)


def test_a_prefix_longer_than_a_sequence_is_masked(device, gx):
    """shared_tokens past a length: the rows of the shorter sequence stop at their own end."""
    rng = np.random.default_rng(8)
    p = Problem(rng, *A, 32, [320, 320], 1, 320)
    p.lengths = [320, 100]
    p.rows[1] = [x[:101] for x in p.rows[1]]
    say("short sequence")
    p.check(p.run(gx))
    p.lengths = [100, 320]                                    # and where the first is the short one
    p.rows = [[x[:101] for x in p.rows[0]], [np.concatenate([p.rows[0][i][:320], p.k[1, p.table[1, 10], :1] if i == 0 else p.v[1, p.table[1, 10], :1]]) for i in range(2)]]
    p.check(p.run(gx))


def test_long_contexts_and_many_splits(device, gx):
    rng = np.random.default_rng(9)
    p = Problem(rng, 10, 2, 128, 64, [20000, 20050], 1, 15000)
    say("long context")
    p.check(p.run(gx))


def test_pools_past_32_bit_offsets(device, gx):
    """Pages whose rows lie more than 2^32 bytes and 2^32 elements into a pool."""
    import torch
    q_heads, kv_heads, d, page = 8, 8, 128, 4096
    layers, pages = 2, 520                                    # 2 x 520 x 4096 x 1024 halves: 8.7 GB a pool
    k, v = (torch.zeros((layers, pages, page, kv_heads, d), dtype=torch.float16, device="cuda") for _ in range(2))
    rng = np.random.default_rng(10)
    n = 5000
    rows = [rng.standard_normal((n + 1, kv_heads, d)).astype(np.float16) for _ in range(2)]
    table = np.array([[519, 517]], np.int32)
    lengths = dev(np.array([0], np.int32))
    references = torch.zeros(pages, dtype=torch.int32, device="cuda")
    t = dev(table)
    cache = gx.KvPages.of(k, v, t, lengths, references)
    say("32-bit offsets")
    gx.launch_kv_pages_append(cache, 1, dev(rows[0][None]), dev(rows[1][None].astype(np.float32)), [0], n + 1)
    gx.launch_kv_pages_advance(cache, [0], n)
    p = Problem(rng, q_heads, kv_heads, d, page, [n], 1, 0)
    p.rows = [rows]
    query, gate = dev(p.query), dev(p.gate)
    out = torch.zeros((1, 1, q_heads, d), dtype=torch.float16, device="cuda")
    work = torch.zeros(gx.kv_pages_attention_workspace_bytes(cache, 1, 1, q_heads, 0), dtype=torch.uint8, device="cuda")
    gx.launch_kv_pages_gated_attention(cache, 1, query, gate, out, [0], 1, q_heads, 0, work)
    p.check(host(out))
    assert float(k[0].abs().max()) == 0.0


def test_results_repeat_and_replay(device, gx):
    """The same bits on every call, on another stream and from a graph replayed as lengths grow."""
    import torch
    rng = np.random.default_rng(11)
    q_heads, kv_heads, d = B
    p = Problem(rng, *B, 16, [100, 120, 97], 3, 96)
    say("repeat")
    first = p.run(gx)
    p.check(first)
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert np.array_equal(p.run(gx, stream=other).view(np.uint16), first.view(np.uint16))
    lengths = dev(np.array([96, 96, 96, 0], np.int32))
    keep = [dev(x) for x in (p.k, p.v, p.table)]
    cache = gx.KvPages.of(*keep, lengths, dev(p.references))
    query, gate = dev(p.query), dev(p.gate)
    out = torch.zeros((3, 3, q_heads, d), dtype=torch.float16, device="cuda")
    work = torch.zeros(gx.kv_pages_attention_workspace_bytes(cache, 3, 3, q_heads, 96), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        gx.launch_kv_pages_gated_attention(cache, 1, query, gate, out, [0, 1, 2], 3, q_heads, 96, work)
    goal = [100, 120, 97]
    full = p.rows
    for turn in range(4):
        p.lengths = [96 + (g - 96) * turn // 3 for g in goal]
        p.rows = [[x[:n + 3] for x in rows] for rows, n in zip(full, p.lengths)]
        lengths.copy_(dev(np.array(p.lengths + [0], np.int32)))
        graph.replay()
        p.check(host(out))
    assert np.array_equal(host(out).view(np.uint16), first.view(np.uint16))


ROWS = [(A, 2, 4), (A, 3, 7), (A, 1, 17), (B, 5, 6), (B, 3, 11), (B, 1, 32), (B, 9, 15)]


@pytest.mark.parametrize("own", [1, 33, 64, 65, 128, 130])
@pytest.mark.parametrize("heads,count,tokens", ROWS)
def test_row_counts_at_the_edges_of_tiles(device, gx, heads, count, tokens, own):
    """Row counts around 16, 32 and 128 of a KV head, ends around the blocks and tiles of positions."""
    rng = np.random.default_rng(count * 100 + tokens + own)
    shared = [0, 63, 129, 256][(count + own) % 4]
    lengths = [max(shared, shared + own - tokens + 3 * i) for i in range(count)]
    p = Problem(rng, *heads, 16, lengths, tokens, shared)
    say("edges", heads, count, tokens, shared, own)
    p.check(p.run(gx))


@pytest.mark.parametrize("heads,tokens", [(A, 1), (A, 7), (B, 1), (B, 7)])
def test_a_damaged_length_stays_its_own_fault(device, gx, heads, tokens):
    """A length past the table leads to missing pages, not past the table; the other sequences keep their results."""
    rng = np.random.default_rng(tokens)
    p = Problem(rng, *heads, 32, [100, 90, 131], tokens, 64)
    p.lengths[1] = -1                                         # 2^32 - 1
    say("damaged length", heads, tokens)
    got = p.run(gx)
    p.lengths[1] = 90
    for i in (0, 2):
        want, tol = p.expect(i)
        assert np.all(np.abs(got[i].astype(np.float64) - want) <= tol)


def _with_a_peak(rng, heads, page, lengths, tokens, shared, at, above):
    """Every row's score at position `at` lies `above` nats over the mean of its others, whose own scores spread by one; the
    value there is zero and all others are positive, large enough that the result is a normal fp16 number.  Nothing but the
    small weights carries the result, and no loss among them is made up for by another."""
    p = Problem(rng, *heads, page, lengths, tokens, shared)
    d = heads[2]
    p.query[..., 0] = 8
    size = min(2.0 ** 14, max(1.0, np.exp(above) * 2.0 ** -20))
    values = [(rng.uniform(0.5, 1.5, x[1].shape) * size).astype(np.float16) for x in p.rows]
    for i, rows in enumerate(p.rows):
        rows[0][..., 0] = 0
        rows[0][at] = 0
        rows[0][at, :, 0] = above * math.sqrt(d) / 8
        values[i][:shared] = values[0][:shared]
        rows[1][...] = values[i]
        rows[1][at] = 0
        for j in range(0, len(rows[0]), page):
            for pool, x in zip((p.k, p.v), rows):
                pool[1, p.table[i, j // page], :len(x[j:j + page])] = x[j:j + page]
    return p


@pytest.mark.parametrize("above", [10, 12, 14, 16, 20, 25])
@pytest.mark.parametrize("heads,page,lengths,tokens,shared,at", [
    ((64, 64, 128), 64, [600] * 8, 1, 0, 5),                  # one item a sequence, by positions
    ((64, 64, 128), 64, [600] * 8, 1, 0, 333),
    ((64, 64, 128), 64, [600] * 8, 32, 0, 5),                 # one item a sequence, by rows
    ((64, 64, 128), 64, [600] * 8, 32, 0, 333),
    ((64, 64, 256), 64, [600] * 8, 1, 0, 5),
    ((128, 64, 256), 64, [600] * 8, 17, 0, 333),
    (A, 16, [2100, 2060, 2200], 1, 2048, 3),                  # many items, the peak in the prefix
    (A, 16, [2100, 2060, 2200], 3, 2048, 1000),
    (B, 32, [2100, 2060, 2200], 3, 2048, 3),
    (A, 16, [40, 33], 1, 0, 39),                              # the peak is the last position of the only block
])
def test_small_weights_beside_a_peak_are_kept(device, gx, heads, page, lengths, tokens, shared, at, above):
    at = min(at, min(lengths))
    p = _with_a_peak(np.random.default_rng(at + tokens), heads, page, lengths, tokens, shared, at, above)
    say("peak", heads, lengths[:3], tokens, shared, at, above)
    got = p.run(gx)
    some = [0, len(lengths) - 1]
    p.check(got[some], some)


@pytest.mark.parametrize("heads,lengths,tokens,shared,at,bad", [
    (A, [40, 45], 1, 0, 7, 30),                               # peak and strange position in one block
    (A, [40, 45], 1, 0, 30, 7),
    (A, [700, 650], 1, 0, 3, 600),                            # in blocks of different waves, in different items
    (A, [700, 650], 1, 0, 600, 3),
    (A, [700, 650], 7, 0, 3, 100),                            # by rows
    (A, [700, 650], 7, 0, 640, 3),
    (A, [2300, 2300], 1, 2048, 5, 2100),                      # the prefix and own positions
    (B, [700, 650], 1, 0, 3, 600),
    (B, [700, 650], 7, 0, 3, 600),
    (B, [2300, 2300], 9, 2048, 5, 2100),
])
def test_strange_positions_far_below_the_peak(device, gx, heads, lengths, tokens, shared, at, bad):
    """Scores 120 nats below a row's largest (2^-173 of its weight): a NaN key and strange values still reach the row."""
    q_heads, kv_heads, d = heads
    group = q_heads // kv_heads
    say("far below", heads, lengths, tokens, shared, at, bad)
    p = _with_a_peak(np.random.default_rng(bad), heads, 16, lengths, tokens, shared, at, 120)
    p.put(0, bad, k=np.full((kv_heads, d), np.nan, np.float16))
    got = p.run(gx)
    assert np.isnan(got[0]).all()
    p.check(got[1:], [1])
    p = _with_a_peak(np.random.default_rng(bad), heads, 16, lengths, tokens, shared, at, 120)
    good = p.rows[0][1][bad].copy()
    value = good.copy()
    value[0, 3], value[1, 5], value[2, d - 1] = np.inf, -np.inf, np.nan
    p.put(0, bad, v=value)
    got = p.run(gx)
    assert np.all(got[0, :, :group, 3] == np.inf) and np.all(got[0, :, group:2 * group, 5] == -np.inf)
    assert np.isnan(got[0, :, 2 * group:3 * group, d - 1]).all()
    touched = np.zeros(got.shape[1:], bool)
    for head, dim in ((0, 3), (1, 5), (2, d - 1)):
        touched[:, head * group:(head + 1) * group, dim] = True
    p.put(0, bad, v=good)
    for i in range(2):
        want, tol = p.expect(i)
        fine = ~touched if i == 0 else np.ones_like(touched)
        assert np.all(np.abs(got[i].astype(np.float64) - want)[fine] <= tol[fine])


@pytest.mark.parametrize("page,hole", [(16, 0), (16, 4), (16, 5), (16, 6), (16, 7), (16, 11), (32, 2), (32, 3), (64, 1), (16, -1)])
@pytest.mark.parametrize("shared", [0, 150])
@pytest.mark.parametrize("heads,tokens", [(A, 1), (A, 7), (B, 1), (B, 9)])
def test_positions_of_missing_pages_are_not_seen(device, gx, heads, tokens, shared, page, hole):
    """A page missing in any 16-position part of a tile, in the prefix or in own positions (and the last page, which holds
    the block's own rows), by positions and by rows; the other sequences do not see it if it is not in the prefix."""
    rng = np.random.default_rng(100 * page + hole + tokens)
    p = Problem(rng, *heads, page, [200, 190, 233], tokens, shared)
    say("missing page", heads, tokens, shared, page, hole)
    held = -(-(p.lengths[0] + tokens) // page)
    hole = hole % held
    p.table[0, hole] = [-1, 100000][hole % 2]
    got = p.run(gx)
    gone = np.zeros(p.lengths[0] + tokens, bool)
    gone[hole * page:(hole + 1) * page] = True
    for i in range(3):
        rows, length = p.rows[i], p.lengths[i]
        for t in range(tokens):
            n = length + t + 1
            keep = np.ones(n, bool)
            if i == 0:
                keep = ~gone[:n]
            else:                                             # the prefix is read through the first sequence's table
                keep[:shared] = ~gone[:shared]
            p.rows[i] = [x[:n][keep] for x in rows]
            p.lengths[i] = int(keep.sum()) - 1 - t
            want, tol = p.expect(i)
            assert np.all(np.abs(got[i, t].astype(np.float64) - want[t]) <= tol[t]), (i, t)
        p.rows[i], p.lengths[i] = rows, length


@pytest.mark.parametrize("heads,tokens", [(A, 1), (A, 7), (B, 1), (B, 9)])
def test_a_sequence_keeps_its_bits_whatever_the_others_hold(device, gx, heads, tokens):
    """Other sequences' queries, own rows (peaks, infinities and NaN among them) and lengths do not change a result's bits."""
    rng = np.random.default_rng(tokens)
    q_heads, kv_heads, d = heads
    lengths = [700, 650, 800, 655]
    p = Problem(rng, *heads, 16, lengths, tokens, 600)
    say("bits", heads, tokens)
    first = p.run(gx)
    p.check(first)
    for i in (0, 3):
        p.query[i] = rng.standard_normal(p.query[i].shape) * 30
        for at in range(600, lengths[i] + tokens):
            k, v = (rng.standard_normal((kv_heads, d)).astype(np.float16) * np.float16(s) for s in (8, 100))
            p.put(i, at, k=k, v=v)
    p.put(3, 610, v=np.full((kv_heads, d), np.inf, np.float16))
    p.put(0, 620, k=np.full((kv_heads, d), np.nan, np.float16))
    p.query[3, 0, 1] = np.nan
    p.lengths[3] = 640
    got = p.run(gx)
    assert not np.array_equal(got[0], first[0])
    for i in (1, 2):
        assert np.array_equal(got[i].view(np.uint16), first[i].view(np.uint16)), i


@pytest.mark.parametrize("shape", ["falling", "rising", "waves", "steps", "wide", "two peaks"])
@pytest.mark.parametrize("heads,lengths,tokens,shared", [
    ((64, 64, 128), [600] * 8, 1, 0), ((64, 64, 128), [600] * 8, 20, 0), ((128, 64, 256), [600] * 4, 17, 0),
    (A, [2100, 2060, 2200], 1, 2048), (B, [2100, 2060, 2200], 3, 2048)])
def test_maxima_that_move_both_ways(device, gx, heads, lengths, tokens, shared, shape):
    """Scores that drift by up to 60 nats along the context, so that a row's stored maximum moves again and again, up, down and
    to the end of its span; values as much larger as scores are lower, as far as fp16 goes."""
    rng = np.random.default_rng(tokens + shared)
    d = heads[2]
    p = Problem(rng, *heads, 16, lengths, tokens, shared)
    p.query[..., 0] = 8
    drift = {"falling": lambda x: -60 * x, "rising": lambda x: 60 * x, "waves": lambda x: 15 * np.sin(40 * x),
             "steps": lambda x: -20 * np.floor(3 * x), "wide": lambda x: 8 * rng.standard_normal(x.shape),
             "two peaks": lambda x: 24.0 * (x == x[3]) + 12.0 * (x == x[len(x) // 2])}[shape]
    for i, rows in enumerate(p.rows):
        n = len(rows[0])
        if i == 0 or not shared:
            high = drift(np.arange(n) / n)
        else:
            high = np.concatenate([first[:shared], drift(np.arange(n) / n)[shared:]])
        first = high if i == 0 else first
        rows[0][..., 0] = (high * math.sqrt(d) / 8)[:, None]
        gain = np.minimum(np.exp(high.max() - high), 2.0 ** 13)
        rows[1][...] = np.clip(rows[1].astype(np.float64) * gain[:, None, None], -60000, 60000)
        if shared and i:
            rows[1][:shared] = p.rows[0][1][:shared]
        for j in range(0, n, 16):
            for pool, x in zip((p.k, p.v), rows):
                pool[1, p.table[i, j // 16], :len(x[j:j + 16])] = x[j:j + 16]
    say("moving maxima", shape, heads, tokens, shared)
    got = p.run(gx)
    some = [0, len(lengths) - 1]
    p.check(got[some], some)
