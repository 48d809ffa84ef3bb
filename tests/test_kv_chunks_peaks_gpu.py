"""Chunk attention where one score stands far above a row's others and its value is zero: the small weights carry the result.

Tolerance, in addition to that of test_kv_chunks_gpu.py (e: a score and its exponential): a weight is rounded to fp16, off by 2^-11 of
itself or, if that is more, by 2^-25 where the row's largest is 2^11 or more.  The weights beside the largest (the zero-valued peaks
here) lose at most 2^-7 of their sum by that 2^-25: where they do not make 2^-18 on average they are held apart.  2^-126 of the
largest is counted as nothing.  Where a tile has at most 32 rows a weight is an fp16 pair, off by 2^-22 of itself or by 2^-25.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

from gpu_util import dev, host, say
from test_kv_chunks_gpu import A, B, U, Chunks

pytestmark = pytest.mark.gpu


def _with_peaks(rng, heads, page, lengths, tokens, peaks, **more):
    """Scores that spread by one nat; at the positions `peaks` (of every sequence) they lie that many nats above, with values of
    zero.  The other values are positive and large enough that the result is a normal fp16 number, so no loss among the small
    weights is made up for by another."""
    c = Chunks(rng, heads, page, lengths, tokens, **more)
    kv_heads, d = heads[1:]
    c.query[..., 0] = 8
    size = min(2.0 ** 14, max(1.0, np.exp(max(peaks.values())) * 2.0 ** -20))
    for i in range(len(lengths)):
        k, v = (x.copy() for x in c.rows[i])
        k[..., 0] = 0
        v[:] = (rng.uniform(0.5, 1.5, v.shape) * size).astype(np.float16)
        for at, above in peaks.items():
            k[at], v[at] = 0, 0
            k[at, :, 0] = above * math.sqrt(d) / 8
        for j in range(len(k)):
            c.put(i, j, k[j], v[j])
    return c


def _check(c, got, sums, which=None, step=2.0 ** -11):
    q_heads, kv_heads, d = c.heads
    for i in range(len(c.tokens)) if which is None else which:
        at, t = c.first(i), c.tokens[i]
        for head in range(q_heads):
            s, size, v = c.rows_of(i, head)
            n = s.shape[1]
            top = s.max(1, keepdims=True)
            w = np.exp(s - top)
            total = w.sum(1, keepdims=True)
            w /= total
            e = (d + 8) * U * size.max(1)[:, None] + 2.0 ** -21
            g = 1 / (1 + np.exp(-c.gate[at:at + t, head, d:].astype(np.float64))) if c.gate is not None else 1.0
            want = w @ v * g
            size = np.abs(v)
            rest = (w * size.any(1)).sum(1, keepdims=True) * size.max(0)
            most = w.max(1, keepdims=True)
            lost = np.minimum(2.0 ** -7 * rest, np.minimum(w, 2.0 ** -36 * most) @ size)
            tol = ((2 * e + step + (n / 2 + 64) * U) * (w @ size) + lost + 2.0 ** -126 * most * size.sum(0)) * g
            tol += np.maximum(np.abs(want) * 2.0 ** -11, 2.0 ** -25) * (1 + 2.0 ** -9)
            off = np.abs(got[at:at + t, head].astype(np.float64) - want)
            assert np.all(off <= tol), (i, head, float(np.max(off / tol)))
            L = top[:, 0] + np.log(total[:, 0])
            off = np.abs(sums[at:at + t, head].astype(np.float64) - L)
            assert np.all(off <= e[:, 0] + (n / 2 + 64) * U + 8 * U * (np.abs(L) + 16)), (i, head, off.max())


@pytest.mark.parametrize("above", [10, 14, 16, 20, 25, 28])
@pytest.mark.parametrize("heads,page,lengths,tokens,at,gap", [
    ((64, 64, 128), 64, [600] * 8, [1] * 8, 5, 1),            # few rows: 512 items of one range
    ((64, 64, 128), 64, [600] * 8, [1] * 8, 333, 1),
    ((64, 64, 128), 64, [600] * 8, [40] * 8, 5, 1),           # many rows, one range
    ((64, 64, 128), 64, [600] * 8, [40] * 8, 333, 1),
    ((64, 64, 256), 64, [600] * 4, [1] * 4, 5, 1),
    ((64, 64, 256), 64, [600] * 4, [40] * 4, 333, 1),
    (A, 16, [2100, 600], [1, 3], 3, 1),                       # many ranges
    (A, 16, [2100, 600], [30, 40], 599, 1),
    (B, 32, [2100, 600], [30, 2], 3, 1),
    (A, 16, [600], [64], 3, 200),                             # ranges of two steps
    (A, 16, [40, 33], [1, 9], 33, 1),                         # the peak is among the last positions
    (B, 16, [40, 33], [1, 9], 33, 1),
])
def test_small_weights_beside_a_peak_are_kept(device, gx, heads, page, lengths, tokens, at, gap, above):
    c = _with_peaks(np.random.default_rng(at + sum(tokens)), heads, page, lengths, tokens, {at: above}, gap=gap)
    say("peak", heads, lengths[:2], tokens[:2], at, above, gap)
    got, sums = c.run(gx)
    _check(c, got, sums, [0, len(lengths) - 1])


@pytest.mark.parametrize("above", [14, 18, 24, 28])
@pytest.mark.parametrize("heads,lengths,tokens,at", [
    ((64, 64, 128), [900] * 8, [1] * 8, [0, 1, 2, 3]),        # side by side
    ((64, 64, 128), [900] * 8, [1] * 8, [10, 140, 270]),      # in blocks that follow each other in a wave
    ((64, 64, 128), [900] * 8, [40] * 8, [10, 70, 140]),      # in steps that follow each other
    ((64, 64, 128), [900] * 8, [40] * 8, [200, 10, 899]),     # apart
    ((64, 64, 256), [900] * 4, [1] * 4, [10, 140, 270]),
    ((64, 64, 256), [900] * 4, [40] * 4, [10, 40, 70]),
    ((64, 64, 256), [900] * 4, [40] * 4, [200, 10, 899]),
])
def test_small_weights_beside_several_peaks_are_kept(device, gx, heads, lengths, tokens, at, above):
    """Peaks of the same height, wherever the others are: in a step that finds its maximum where it was before, too."""
    c = _with_peaks(np.random.default_rng(sum(at)), heads, 64, lengths, tokens, dict.fromkeys(at, above))
    say("peaks", heads, tokens[0], at, above)
    got, sums = c.run(gx)
    _check(c, got, sums, [0, len(lengths) - 1])


@pytest.mark.parametrize("heads", [A, B])
@pytest.mark.parametrize("tokens", [1, 40])
def test_scores_that_fall_and_rise_by_much(device, gx, heads, tokens):
    """Steps whose largest scores lie 10 to 60 nats apart, up and down."""
    q_heads, kv_heads, d = heads
    rng = np.random.default_rng(17 + tokens)
    for levels in ([0, 30, 0, 12, 45, 5], [60, 0, 20, 59, 1, 30], [0, -40, 10, -20, 25, 24]):
        c = _with_peaks(rng, heads, 32, [6 * 160], [tokens], {0: 1.0})
        for j in range(6 * 160):
            k = c.rows[0][0][j].copy()
            k[:, 0] = levels[j // 160] * math.sqrt(d) / 8
            c.put(0, j, k=k, v=rng.standard_normal((kv_heads, d)).astype(np.float16))
        say("levels", heads, tokens, levels)
        got, sums = c.run(gx)
        _check(c, got, sums)


@pytest.mark.parametrize("heads,tokens,at,bad", [
    (A, 1, 7, 30), (A, 1, 30, 7), (A, 1, 3, 600), (A, 40, 3, 100), (A, 40, 640, 3), (A, 40, 30, 7), (B, 1, 3, 600), (B, 40, 3, 600),
])
def test_strange_positions_far_below_the_peak(device, gx, heads, tokens, at, bad):
    """Scores 120 nats below a row's largest: a NaN key and strange values still reach the rows that see them, and no others."""
    q_heads, kv_heads, d = heads
    group = q_heads // kv_heads
    say("far below", heads, tokens, at, bad)

    def make():
        return _with_peaks(np.random.default_rng(bad), heads, 16, [700, 650], [tokens] * 2, {at: 120})

    c = make()
    c.put(0, bad, k=np.full((kv_heads, d), np.nan, np.float16))
    got, sums = c.run(gx)
    assert np.isnan(got[:tokens]).all() and np.isnan(sums[:tokens]).all()
    _check(c, got, sums, [1])
    c = make()
    good = c.rows[0][1][bad].copy()
    value = good.copy()
    value[0, 3], value[1, 5], value[2, d - 1] = np.inf, -np.inf, np.nan
    c.put(0, bad, v=value)
    got, sums = c.run(gx)
    got = got.copy()
    assert np.all(got[:tokens, :group, 3] == np.inf) and np.all(got[:tokens, group:2 * group, 5] == -np.inf)
    assert np.isnan(got[:tokens, 2 * group:3 * group, d - 1]).all()
    c.put(0, bad, v=good)
    for head, dim in ((0, 3), (1, 5), (2, d - 1)):            # the rest is as without them
        for h in range(head * group, head * group + group):
            s, _, v = c.rows_of(0, h)
            w = np.exp(s - s.max(1, keepdims=True))
            got[:tokens, h, dim] = (w @ v[:, dim]) / w.sum(1) / (1 + np.exp(-c.gate[:tokens, h, d + dim].astype(np.float64)))
    _check(c, got, sums)


@pytest.mark.parametrize("heads,lengths,tokens", [(A, [600, 33, 0, 2100], [1, 3, 6, 2]), (B, [700, 31, 0, 2100], [1, 5, 2, 3])])
def test_few_rows_carry_their_weights_in_pairs(device, gx, heads, lengths, tokens):
    """Equal values but for a sign, so that nearly all of the output cancels and what is left is a normal fp16 number."""
    rng = np.random.default_rng(sum(tokens))
    c = Chunks(rng, heads, 16, lengths, tokens)
    for i, n in enumerate(lengths):
        v = c.rows[i][1]
        v[:] = np.where(rng.random(v.shape) < 0.5, 1, -1).astype(np.float16)
        for j in range(len(v)):
            c.put(i, j, v=v[j])
    say("pairs", heads, lengths, tokens)
    got, sums = c.run(gx)
    _check(c, got, sums, None, 2.0 ** -22)


@pytest.mark.parametrize("heads", [A, B])
def test_a_prompt_whose_first_rows_see_few_positions(device, gx, heads):
    """Rows of one position, of two that lie 30 nats apart, and so on, beside rows that see hundreds."""
    c = _with_peaks(np.random.default_rng(18), heads, 16, [0, 1], [300, 2], {0: 30})
    say("first rows", heads)
    c.query[1::2, :, 0] = 0                                    # every other row has no peak
    got, sums = c.run(gx)
    _check(c, got, sums)
