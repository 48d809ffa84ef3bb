"""Ragged chunk attention over K/V pages, and the weight that cached rows receive, on the GPU against 64 bits.

Tolerances.  u = 2^-24 is half a step of fp32.  A score is a sum of D products accumulated in fp32: off by at most
D u |q|.|k| / sqrt(D), and scaling, the difference to the maximum and the exponential add a few u of the score and 2^-21 of the
weight: e = (D + 8) u max(|q|.|k|) / sqrt(D) + 2^-21 in all, once for the score and once for the maximum.
- A weight goes into the second product in fp16, scaled so that the row's largest is 2^11 or more: half a step is 2^-11 of it,
  and 2^-25 below 2^-14, 2^-36 of the largest.  Sums over n positions add (n / 2 + 64) u.  The result is rounded to fp16 once
  (2^-11 of it, 2^-25 below the normal numbers).
- The log of the sum is off by e, by the sum's (n / 2 + 64) u, and by a few u of itself and of the lift of 11 binades.
- A received weight is exp(score - L) for given L: e plus 8 u (|score| + |L| + 4) of each, and the additions, rows / 2 at most in
  a row of them.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

from gpu_util import dev, host, say

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
A, B = (40, 8, 128), (24, 4, 256)


class Chunks:
    """Two layers of pages in no order; what no sequence sees is NaN: rows past the ends, free pages, layer 0."""

    def __init__(self, rng, heads, page, lengths, tokens, gate=True, slack=2, spread=1.0, gap=1):
        q_heads, kv_heads, d = self.heads = heads
        self.page, self.lengths, self.tokens = page, list(lengths), list(tokens)
        held = [-(-(n + t) // page) for n, t in zip(lengths, tokens)]
        pages = sum(held) + slack
        order = rng.permutation(pages).tolist()
        self.k, self.v = (np.full((2, pages, page, kv_heads, d), np.nan, np.float16) for _ in range(2))
        self.table = np.full((len(lengths) + 1, max(held) + gap), -1, np.int32)
        self.references, self.rows, at = np.zeros(pages, np.int32), [], 0
        for i, h in enumerate(held):
            mine = order[at:at + h]
            at += h
            self.table[i, :h] = mine
            self.references[mine] = 1
            kv = [(rng.standard_normal((lengths[i] + tokens[i], kv_heads, d)) * spread).astype(np.float16) for _ in range(2)]
            self.rows.append(kv)
            for pool, x in zip((self.k, self.v), kv):
                for j in range(0, len(x), page):
                    pool[1, mine[j // page], :len(x[j:j + page])] = x[j:j + page]
        self.hidden = [np.zeros(n + t, bool) for n, t in zip(lengths, tokens)]      # positions without a page
        self.query = rng.standard_normal((sum(tokens), q_heads, d)).astype(np.float16)
        self.gate = (rng.standard_normal((sum(tokens), q_heads, 2 * d)) * 2).astype(np.float32) if gate else None
        if gate:
            self.gate[..., :d] = np.nan                       # the query half of the projection is not read

    def put(self, i, position, k=None, v=None):
        """Overwrites rows of one position of one sequence, in its page and in the reference."""
        for pool, rows, x in ((self.k, self.rows[i][0], k), (self.v, self.rows[i][1], v)):
            if x is not None:
                rows[position] = x
                pool[1, self.table[i, position // self.page], position % self.page] = x

    def lose(self, i, column):
        self.table[i, column] = -1
        self.hidden[i][column * self.page:(column + 1) * self.page] = True

    def first(self, i):
        return sum(self.tokens[:i])

    def pages(self, gx):
        self.device = [dev(x) for x in (self.k, self.v, self.table, np.array(self.lengths + [0], np.int32), self.references)]
        return gx.KvPages.of(*self.device)

    def run(self, gx, sums=True, stream=None, listed=None):
        """Outputs and log sums, rows behind the last one checked to be as they were."""
        import torch
        q_heads, kv_heads, d = self.heads
        pages, rows = self.pages(gx), sum(self.tokens)
        out = torch.full((rows + 1, q_heads, d), 7.0, dtype=torch.float16, device="cuda")
        log_sums = torch.full((rows + 1, q_heads), 7.0, device="cuda") if sums else None
        work = torch.full((max(16, gx.kv_pages_chunk_attention_workspace_bytes(pages, self.tokens, q_heads)),), 0xff, dtype=torch.uint8,
                          device="cuda")
        gate = dev(self.gate) if self.gate is not None else None
        gx.launch_kv_pages_chunk_attention(pages, 1, dev(self.query), gate, out, log_sums,
                                           range(len(self.tokens)) if listed is None else listed, self.tokens, q_heads, work, stream=stream)
        got, got_sums = host(out), host(log_sums) if sums else np.full((rows + 1, q_heads), 7.0)
        assert np.all(got[-1] == 7.0) and np.all(got_sums[-1] == 7.0)
        return got[:-1], got_sums[:-1]

    def rows_of(self, i, head):
        """Scores [tokens, positions] with -inf where unseen, |q|.|k| / sqrt(D), values, in 64 bits."""
        q_heads, kv_heads, d = self.heads
        n, t = self.lengths[i], self.tokens[i]
        at = self.first(i)
        q = self.query[at:at + t, head].astype(np.float64)
        k, v = (x[:, head // (q_heads // kv_heads)].astype(np.float64) for x in self.rows[i])
        unseen = (np.arange(n + t) > n + np.arange(t)[:, None]) | self.hidden[i]
        with np.errstate(invalid="ignore", over="ignore"):
            s = np.where(unseen, -np.inf, q @ k.T / math.sqrt(d))
            return s, np.where(unseen, 0, np.abs(q) @ np.abs(k).T / math.sqrt(d)), v

    def check(self, got, sums=None, which=None):
        q_heads, kv_heads, d = self.heads
        for i in range(len(self.tokens)) if which is None else which:
            at, t = self.first(i), self.tokens[i]
            for head in range(q_heads):
                s, size, v = self.rows_of(i, head)
                n = s.shape[1]
                top = s.max(1, keepdims=True, initial=-np.inf)
                empty = top[:, 0] == -np.inf
                w = np.exp(s - np.where(empty[:, None], 0, top))
                total = w.sum(1, keepdims=True)
                w /= np.where(total == 0, 1, total)
                e = (d + 8) * U * size.max(1, initial=0)[:, None] + 2.0 ** -21
                g = 1 / (1 + np.exp(-self.gate[at:at + t, head, d:].astype(np.float64))) if self.gate is not None else 1.0
                want = w @ v * g
                tol = ((2 * e + 2.0 ** -11 + (n / 2 + 64) * U) * (w @ np.abs(v)) + 2.0 ** -36 * w.max(1, keepdims=True, initial=0) * np.abs(v).sum(0)) * g
                tol += np.maximum(np.abs(want) * 2.0 ** -11, 2.0 ** -25) * (1 + 2.0 ** -9)
                off = np.abs(got[at:at + t, head].astype(np.float64) - want)
                assert np.all(off <= tol), (i, head, float(np.max(off / tol)))
                if sums is not None:
                    L = np.where(empty, -np.inf, top[:, 0] + np.log(np.where(empty, 1, total[:, 0])))
                    x = sums[at:at + t, head].astype(np.float64)
                    assert np.array_equal(x == -np.inf, empty)
                    off = np.abs(np.where(empty, 0, x) - np.where(empty, 0, L))
                    assert np.all(off <= e[:, 0] + (n / 2 + 64) * U + 8 * U * (np.abs(np.where(empty, 0, L)) + 16)), (i, head, off.max())


CASES = [
    ((1, 1, 128), 16, [0], [1]),                              # one position: the token itself
    ((1, 1, 256), 16, [0, 1, 2], [1, 1, 1]),
    ((2, 1, 128), 16, [0, 15, 16, 17, 31, 32, 33, 63, 64, 65], [1, 2, 1, 3, 1, 2, 1, 1, 2, 1]),
    ((6, 2, 128), 32, [5, 0, 40], [0, 3, 0]),                 # sequences without rows
    ((16, 1, 128), 16, [100, 130], [8, 9]),                   # 128 rows, a full tile, and 144
    ((17, 1, 128), 64, [0, 61], [8, 70]),
    (A, 16, [0], [300]),                                      # a prompt from the start
    (A, 64, [509, 0, 1200, 77], [1, 130, 1, 26]),             # chunks beside decoding sequences
    (A, 256, [2100] * 5, [1, 1, 1, 1, 2]),
    (A, 16, list(range(40, 73)), [1 + i % 3 for i in range(33)]),
    (A, 128, [3000], [150]),
    (B, 16, [0], [111]),
    (B, 32, [200, 1300, 201], [5, 70, 1]),
    (B, 4096, [5000, 4090], [2, 9]),                          # pages longer than a range
    (B, 64, [129, 257, 31, 32, 33], [32, 1, 1, 1, 1]),
    ((8, 8, 128), 16, [700, 3], [140, 2]),                    # no grouping
    ((24, 3, 256), 16, list(range(1, 20)), [3] * 19),
    ((5, 5, 128), 32, [64] * 256, [1] * 256),                 # as many sequences as a call takes
]


@pytest.mark.parametrize("heads,page,lengths,tokens", CASES)
@pytest.mark.parametrize("gate", [True, False])
def test_attention_equals_the_definition(device, gx, heads, page, lengths, tokens, gate):
    rng = np.random.default_rng(len(lengths) * 1000 + page + sum(tokens))
    c = Chunks(rng, heads, page, lengths, tokens, gate)
    say("chunk attention", heads, page, lengths[:6], tokens[:6], gate)
    got, sums = c.run(gx, sums=gate)
    c.check(got, sums if gate else None)


@pytest.mark.parametrize("heads,page,lengths,tokens", [((32, 1, 256), 32, [100, 60], [1050, 1]), ((32, 1, 128), 64, [300, 5], [2070, 2])])
def test_more_tiles_than_places(device, gx, heads, page, lengths, tokens):
    """Tiles that are not divided beside a rest that is, a decoding sequence's few rows among them."""
    c = Chunks(np.random.default_rng(sum(tokens)), heads, page, lengths, tokens)
    say("more tiles than places", heads, page, lengths, tokens)
    c.check(*c.run(gx))


@pytest.mark.parametrize("heads", [A, B])
def test_a_wide_table_divides_the_positions(device, gx, heads):
    """The same rows with a table that leaves room: other ranges, the same result within its tolerance."""
    rng = np.random.default_rng(4)
    say("wide table", heads)
    for gap in (1, 200):
        c = Chunks(rng, heads, 32, [1000, 3, 517], [40, 7, 1], gap=gap)
        got, sums = c.run(gx)
        c.check(got, sums)


@pytest.mark.parametrize("heads", [A, B])
@pytest.mark.parametrize("spread", [0.02, 4.0, 30.0])
def test_scores_that_hardly_differ_and_that_differ_much(device, gx, heads, spread):
    rng = np.random.default_rng(8)
    c = Chunks(rng, heads, 16, [400, 60], [20, 33], spread=spread)
    say("spread of scores", heads, spread)
    got, sums = c.run(gx)
    c.check(got, sums)


@pytest.mark.parametrize("heads", [A, B])
def test_scores_that_climb_along_the_context(device, gx, heads):
    """Every tile has a new maximum, or every tile lies below the first."""
    q_heads, kv_heads, d = heads
    for way in (1, -1):
        rng = np.random.default_rng(9)
        c = Chunks(rng, heads, 16, [500], [64])
        c.query[:] = np.abs(c.query)
        climb = np.linspace(-1, 1, 564)[:, None, None] * way
        for j in range(564):
            c.put(0, j, k=(np.abs(c.rows[0][0][j]) * climb[j]).astype(np.float16))
        say("climbing scores", heads, way)
        got, sums = c.run(gx)
        c.check(got, sums)


@pytest.mark.parametrize("heads", [A, B])
def test_a_peak_far_above_the_others(device, gx, heads):
    """One score 16 nats above the rest, its value zero: the rest carry the output."""
    q_heads, kv_heads, d = heads
    rng = np.random.default_rng(10)
    c = Chunks(rng, heads, 32, [600], [4], spread=0.05)
    c.query[:] = np.float16(1.0) + (rng.random(c.query.shape) * 0.01).astype(np.float16)
    c.put(0, 300, k=np.full((kv_heads, d), 16 / math.sqrt(d), np.float16), v=np.zeros((kv_heads, d), np.float16))
    say("peak", heads)
    got, sums = c.run(gx)
    c.check(got, sums)


@pytest.mark.parametrize("heads", [A, B])
@pytest.mark.parametrize("wide", [False, True])
def test_infinities_and_nan_reach_the_rows_that_see_them(device, gx, heads, wide):
    """Among the chunk's own rows: earlier tokens do not see them, whatever the positions are divided into."""
    q_heads, kv_heads, d = heads
    rng = np.random.default_rng(12)
    lengths, tokens = [300, 90], [40, 6]
    for value in (np.inf, -np.inf, np.nan):
        c = Chunks(rng, heads, 16, lengths, tokens, gap=200 if wide else 1)
        v = c.rows[0][1][317].copy()
        v[0, 5] = value
        c.put(0, 317, v=v)                                    # seen by tokens 17.. of KV head 0
        k = c.rows[1][0][93].copy()
        k[kv_heads - 1, 3] = np.nan
        c.put(1, 93, k=k)                                     # seen by tokens 3.. of the last KV head
        say("strange values", heads, wide, value)
        got, sums = c.run(gx)
        group = q_heads // kv_heads
        first = got[17:40, :group, 5].astype(np.float64)
        assert np.all(np.isnan(first) if np.isnan(value) else first == value)
        assert np.isnan(got[43:, -group:]).all() and np.isnan(sums[43:, -group:]).all()
        # Everything else is as without them.
        for s, j, pool, head, e in ((0, 317, 1, 0, 5), (1, 93, 0, kv_heads - 1, 3)):
            c.rows[s][pool][j, head, e] = 0.0
        got, sums = got.copy(), sums.copy()
        want = Chunks.__new__(Chunks)
        want.__dict__.update(c.__dict__)
        clean = np.zeros_like(got)
        got[17:40, :group, 5], got[43:, -group:], sums[43:, -group:] = 0, 0, 0
        # The masked-out places are taken from the definition itself.
        for i in range(2):
            for head in range(q_heads):
                s, _, vv = c.rows_of(i, head)
                w = np.exp(s - s.max(1, keepdims=True))
                w /= w.sum(1, keepdims=True)
                at = c.first(i)
                g = 1 / (1 + np.exp(-c.gate[at:at + c.tokens[i], head, d:].astype(np.float64)))
                clean[at:at + c.tokens[i], head] = w @ vv * g
                L = np.log(np.exp(s - s.max(1, keepdims=True)).sum(1)) + s.max(1)
                if i == 1 and head >= q_heads - group:
                    sums[43:, head] = L[3:]
        got[17:40, :group, 5], got[43:, -group:] = clean[17:40, :group, 5], clean[43:, -group:]
        c.check(got, sums)


@pytest.mark.parametrize("heads", [A, B])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("wide", [False, True])
def test_missing_pages_are_not_seen(device, gx, heads, page, wide):
    rng = np.random.default_rng(13)
    c = Chunks(rng, heads, page, [700, 5, page], [9, 30, 2], gap=200 if wide else 1)
    c.lose(0, 0)
    c.lose(0, 700 // page - 1)
    c.lose(2, 0)                                              # the tokens of sequence 2 see themselves only
    c.table[1, 0] = len(c.references) + 3                     # an entry that names no page is none
    c.hidden[1][:page] = True                                 # the first tokens of sequence 1 may see nothing
    say("missing pages", heads, page, wide)
    got, sums = c.run(gx)
    c.check(got, sums)
    if page == 64:
        assert np.all(got[9:39] == 0) and np.all(sums[9:39] == -np.inf)


def test_one_sequence_several_times_and_orders(device, gx):
    """A list may name a sequence twice; its order is the order of the rows; a call repeated gives the same bits."""
    rng = np.random.default_rng(14)
    c = Chunks(rng, A, 16, [333, 50], [6, 6])
    say("order of the list")
    got, sums = c.run(gx)
    c.check(got, sums)
    again, again_sums = c.run(gx)
    assert np.array_equal(got, again) and np.array_equal(sums, again_sums)
    query, gate = c.query, c.gate
    swapped = lambda x: np.concatenate([x[6:], x[:6]])  # noqa: E731
    c.query, c.gate = swapped(query), swapped(gate)
    other, other_sums = c.run(gx, listed=[1, 0])
    c.query, c.gate = query, gate
    c.check(swapped(other), swapped(other_sums))
    c.query, c.gate = (np.concatenate([x[:6], x[:6]]) for x in (query, gate))
    twice, twice_sums = c.run(gx, listed=[0, 0])
    c.query, c.gate = query, gate
    for half in (slice(0, 6), slice(6, 12)):
        c.check(np.concatenate([twice[half], got[6:]]), np.concatenate([twice_sums[half], sums[6:]]))


def test_offsets_past_32_bits(device, gx):
    """A pool of more than 2^31 elements: the last page and the last layer's rows are reached."""
    import torch
    kv_heads, d, page = 8, 128, 4096
    pool = torch.zeros(2, 300, page, kv_heads, d, dtype=torch.float16, device="cuda")
    rng = np.random.default_rng(15)
    x = rng.standard_normal((2, 200, kv_heads, d)).astype(np.float16)
    values = torch.zeros_like(pool)
    pool[1, 299, :200], values[1, 299, :200] = dev(x[0]), dev(x[1])
    table, lengths, references = dev(np.array([[299]], np.int32)), dev(np.array([150], np.int32)), torch.ones(300, dtype=torch.int32, device="cuda")
    pages = gx.KvPages.of(pool, values, table, lengths, references)
    c = Chunks(rng, A, 256, [150], [50])
    for j in range(200):
        c.put(0, j, x[0][j], x[1][j])
    out, sums = torch.zeros(50, 40, 128, dtype=torch.float16, device="cuda"), torch.zeros(50, 40, device="cuda")
    work = torch.empty(max(16, gx.kv_pages_chunk_attention_workspace_bytes(pages, [50], 40)), dtype=torch.uint8, device="cuda")
    say("large pool")
    gx.launch_kv_pages_chunk_attention(pages, 1, dev(c.query), dev(c.gate), out, sums, [0], [50], 40, work)
    c.check(host(out), host(sums))


def test_a_damaged_length_stays_in_bounds(device, gx):
    rng = np.random.default_rng(16)
    c = Chunks(rng, A, 16, [100], [3])
    c.lengths[0] = -1                                         # 2^32 - 1 committed tokens
    say("damaged length")
    pages = c.pages(gx)
    c.lengths[0] = 100
    import torch
    out = torch.zeros(4, 40, 128, dtype=torch.float16, device="cuda")
    work = torch.empty(max(16, gx.kv_pages_chunk_attention_workspace_bytes(pages, [3], 40)), dtype=torch.uint8, device="cuda")
    gx.launch_kv_pages_chunk_attention(pages, 1, dev(c.query), None, out, None, [0], [3], 40, work)
    # The rest of the last page, NaN here, counts as committed; nothing else is reached.
    assert np.isnan(host(out)[:3]).all() and not host(out)[3].any()


# ---- the weight that cached rows receive -----------------------------------------------------


def _weights(c, gx, sums, weight, stream=None):
    """Runs the accumulation over what the rows have; [sequences + 1, capacity]."""
    import torch
    pages = c.pages(gx)
    w, p, d = dev(weight), torch.zeros(weight.shape, dtype=torch.int32, device="cuda"), torch.zeros(len(weight), dtype=torch.int32, device="cuda")
    kv = gx.KvWeights.of(pages, w, p, d)
    work = torch.full((gx.kv_weights_workspace_bytes(pages, c.tokens, c.heads[0]),), 0xff, dtype=torch.uint8, device="cuda")
    gx.launch_kv_weights_add(pages, kv, 1, dev(c.query), dev(sums), range(len(c.tokens)), c.tokens, c.heads[0], work, stream=stream)
    assert not host(p).any() and not host(d).any()
    return host(w)


def _check_weights(c, got, sums, before):
    q_heads, kv_heads, d = c.heads
    for i, t in enumerate(c.tokens):
        n, at = c.lengths[i] + t, c.first(i)
        want, tol = before[i, :n].astype(np.float64), np.zeros(n)
        for head in range(q_heads):
            s, size, _ = c.rows_of(i, head)
            L = sums[at:at + t, head].astype(np.float64)[:, None]
            good = np.isfinite(L)
            with np.errstate(invalid="ignore"):
                w = np.where(good & np.isfinite(s), np.exp(np.where(np.isfinite(s), s, 0) - np.where(good, L, 0)), 0)
            e = (d + 8) * U * size + 2.0 ** -21 + 8 * U * (np.abs(np.where(np.isfinite(s), s, 0)) + np.abs(np.where(good, L, 0)) + 4)
            want = want + w.sum(0)
            tol += (w * e).sum(0)
        tol += want * U * (t * q_heads / kv_heads / 2 + 64 + kv_heads)
        off = np.abs(got[i, :n] - want)
        assert np.all(off <= tol), (i, float(np.max(off / tol)))
        assert np.array_equal(got[i, n:], before[i, n:])      # nothing behind the sequence is touched
    assert np.array_equal(got[-1], before[-1])


@pytest.mark.parametrize("heads,page,lengths,tokens", CASES)
def test_weights_equal_the_definition(device, gx, heads, page, lengths, tokens):
    rng = np.random.default_rng(len(lengths) * 1000 + page + sum(tokens))
    c = Chunks(rng, heads, page, lengths, tokens, gate=False)
    say("received weights", heads, page, lengths[:6], tokens[:6])
    sums = np.zeros((sum(tokens), heads[0]), np.float32)
    for i, t in enumerate(tokens):
        for head in range(heads[0]):
            s = c.rows_of(i, head)[0]
            sums[c.first(i):c.first(i) + t, head] = s.max(1, initial=-np.inf) + np.log(np.exp(s - s.max(1, keepdims=True, initial=-np.inf)).sum(1))
    before = (rng.random((len(lengths) + 1, c.table.shape[1] * page)) * 3).astype(np.float32)
    got = _weights(c, gx, sums, before)
    _check_weights(c, got, sums, before)
    assert np.array_equal(got, _weights(c, gx, sums, before))  # the same bits every time


@pytest.mark.parametrize("heads", [(40, 1, 128), (33, 1, 256), (128, 2, 128)])
def test_weights_of_wide_groups(device, gx, heads):
    """More query heads to a KV head than rows are staged at a time: a step lies within a token, or in two."""
    rng = np.random.default_rng(sum(heads))
    c = Chunks(rng, heads, 16, [300, 3, 0], [9, 1, 20], gate=False)
    say("received weights of wide groups", heads)
    got, sums = c.run(gx)
    c.check(got, sums)
    before = rng.random((4, c.table.shape[1] * 16)).astype(np.float32)
    _check_weights(c, _weights(c, gx, sums, before), sums, before)


def test_weights_of_long_caches(device, gx):
    """More positions than a launch has workgroups for: a chunk's (256 each) and a decoding sequence's (32 each)."""
    rng = np.random.default_rng(24)
    c = Chunks(rng, (1, 1, 128), 4096, [262300, 33000], [40, 1], gate=False, gap=0)
    say("received weights of long caches")
    sums = np.zeros((41, 1), np.float32)
    for i, t in enumerate(c.tokens):
        s = c.rows_of(i, 0)[0]
        sums[c.first(i):c.first(i) + t, 0] = s.max(1) + np.log(np.exp(s - s.max(1, keepdims=True)).sum(1))
    before = rng.random((3, c.table.shape[1] * 4096)).astype(np.float32)
    _check_weights(c, _weights(c, gx, sums, before), sums, before)


@pytest.mark.parametrize("heads", [A, B])
def test_weights_of_missing_pages_and_rows_that_see_nothing(device, gx, heads):
    rng = np.random.default_rng(21)
    c = Chunks(rng, heads, 16, [200, 40], [30, 3], gate=False)
    c.lose(0, 3)
    sums = (rng.standard_normal((33, heads[0])) + 5).astype(np.float32)
    sums[4], sums[7, 1] = -np.inf, np.nan                      # rows that add nothing
    before = np.ones((3, c.table.shape[1] * 16), np.float32)
    say("weights of missing pages", heads)
    got = _weights(c, gx, sums, before)
    assert np.array_equal(got[0, 48:64], before[0, 48:64])
    _check_weights(c, got, sums, before)


def test_other_streams_and_devices(device, gx):
    """A call on a stream that is not the current one, and tensors that the call's GPU does not reach."""
    import torch
    rng = np.random.default_rng(22)
    c = Chunks(rng, A, 16, [100, 7], [20, 1])
    say("another stream")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    got, sums = c.run(gx, stream=stream)
    c.check(got, sums)
    pages = c.pages(gx)
    out, cpu = torch.zeros(21, 40, 128, dtype=torch.float16, device="cuda"), torch.zeros(21, 40, 128, dtype=torch.float16)
    work = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    for bad in (lambda: gx.launch_kv_pages_chunk_attention(pages, 1, cpu, None, out, None, [0, 1], [20, 1], 40, work),
                lambda: gx.launch_kv_pages_chunk_attention(pages, 1, out, None, cpu, None, [0, 1], [20, 1], 40, work),
                lambda: gx.launch_kv_pages_chunk_attention(pages, 1, out.float(), None, out, None, [0, 1], [20, 1], 40, work),
                lambda: gx.launch_kv_pages_chunk_attention(pages, 1, out[:20], None, out, None, [0, 1], [20, 1], 40, work)):
        with pytest.raises(ValueError):
            bad()


def test_captured_attention_and_weights_follow_the_device_state(device, gx):
    """Recorded once; lengths, tables and inputs change between the replays."""
    import torch
    rng = np.random.default_rng(23)
    c = Chunks(rng, A, 16, [300, 40], [25, 1])
    pages = c.pages(gx)
    capacity = c.table.shape[1] * 16
    query, gate = dev(c.query), dev(c.gate)
    out, sums = torch.zeros(26, 40, 128, dtype=torch.float16, device="cuda"), torch.zeros(26, 40, device="cuda")
    weight, position, dropped = torch.zeros(3, capacity, device="cuda"), torch.zeros(3, capacity, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    kv = gx.KvWeights.of(pages, weight, position, dropped)
    work = torch.empty(max(16, gx.kv_pages_chunk_attention_workspace_bytes(pages, c.tokens, 40)), dtype=torch.uint8, device="cuda")
    work2 = torch.empty(gx.kv_weights_workspace_bytes(pages, c.tokens, 40), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        gx.launch_kv_pages_chunk_attention(pages, 1, query, gate, out, sums, [0, 1], c.tokens, 40, work)
        gx.launch_kv_weights_add(pages, kv, 1, query, sums, [0, 1], c.tokens, 40, work2)
    for lengths in ([300, 40], [120, 3], [0, 41]):
        short = Chunks.__new__(Chunks)
        short.__dict__.update(c.__dict__)
        short.lengths = lengths
        short.rows = [[x[:n + t] for x in kv_rows] for kv_rows, n, t in zip(c.rows, lengths, c.tokens)]
        short.hidden = [np.zeros(n + t, bool) for n, t in zip(lengths, c.tokens)]
        if lengths[1] == 41:                                  # one more row than the sequence was made with
            row = [rng.standard_normal((1, 8, 128)).astype(np.float16) for _ in range(2)]
            for pool, x in zip(c.device[:2], row):
                pool[1, int(c.table[1, 41 // 16]), 41 % 16] = dev(x[0])
            short.rows[1] = [np.concatenate([a[:41], b]) for a, b in zip(c.rows[1], row)]
        c.device[3][:2] = dev(np.array(lengths, np.int32))
        weight.fill_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        got, got_sums = host(out), host(sums)
        short.check(got, got_sums)
        _check_weights(short, host(weight), got_sums, np.full((3, capacity), 0.5, np.float32))
