"""Logit rules on the GPU against the formula in 64 bits.

Tolerance: the rules are at most five fp32 operations after another, each off by at most half a step (2^-24 of its
result), so an output is within 2^-24 (1 + 2^-20) of the sum of the magnitudes of the intermediate results.  Tokens are
compared with the argmax of the launcher's own output: exact.
"""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import dev, empty, host, say

pytestmark = pytest.mark.gpu
HALF_STEP = 2.0 ** -24 * (1 + 2.0 ** -20)


def _problem(rng, batch, vocabulary, history=0, bias=0, masks=0, rows=None):
    """Arrays by the names of gfxinfer_logit_rules."""
    a = {}
    if history:
        n = batch if rows is None else rows
        a["history"] = (rng.random((n, history)) ** 4 * (vocabulary * 1.05)).astype(np.uint32)   # some past the vocabulary
        a["history"][0, 0] = 0xffffffff
        a["history_lengths"] = rng.integers(0, history + 3, batch).astype(np.uint32)              # clamped to the row
        a["prompt_lengths"] = rng.integers(0, history + 1, batch).astype(np.uint32)
        a["repetition"] = (1 + rng.random(batch) * 0.5).astype(np.float32)
        a["presence"], a["frequency"] = (rng.random(batch).astype(np.float32) for _ in range(2))
        if rows is not None:
            a["history_rows"] = rng.integers(-1, rows + 1, batch).astype(np.int32)
    if bias:
        a["bias_tokens"] = (rng.random((batch, bias)) ** 2 * vocabulary * 1.1).astype(np.uint32)  # repeated tokens too
        a["bias_values"] = (rng.standard_normal((batch, bias)) * 5).astype(np.float32)
        a["bias_counts"] = rng.integers(0, bias + 1, batch).astype(np.uint32)
    if masks:
        a["allowed"] = rng.integers(0, 1 << 32, (masks, (vocabulary + 31) // 32), dtype=np.uint64).astype(np.uint32)
        a["allowed_rows"] = rng.integers(-1, masks + 1, batch).astype(np.int32)
    return a


def _formula(logits, a):
    """(result, sum of the magnitudes of the intermediate results), both fp64."""
    batch, vocabulary = logits.shape
    out, size = logits.astype(np.float64), np.zeros(logits.shape)
    with np.errstate(all="ignore"):
        for b in range(batch):
            x = out[b]
            row = int(a["history_rows"][b]) if "history_rows" in a else b
            if "history" in a and 0 <= row < len(a["history"]):
                tokens = a["history"][row][:a["history_lengths"][b]].astype(np.int64)
                prompt = int(a["prompt_lengths"][b]) if "prompt_lengths" in a else 0
                seen, count = (np.bincount(t[t < vocabulary], minlength=vocabulary) for t in (tokens, tokens[prompt:]))
                factor, f, p = (float(a[k][b]) if k in a else d for k, d in (("repetition", 1), ("frequency", 0), ("presence", 0)))
                x = np.where(seen > 0, np.where(x > 0, x / factor, x * factor), x)
                size[b] += np.abs(x) + 2 * f * count
                x = x - f * count
                size[b] += np.abs(x)
                x = np.where(count > 0, x - p, x)
                size[b] += np.abs(x)
            if "bias_tokens" in a:
                n = int(a["bias_counts"][b]) if "bias_counts" in a else a["bias_tokens"].shape[1]
                added = {int(t): float(v) for t, v in zip(a["bias_tokens"][b][:n], a["bias_values"][b][:n]) if t < vocabulary}
                x = x.copy()
                for t, v in added.items():
                    x[t] += v
                size[b] += np.abs(x)
            row = int(a["allowed_rows"][b]) if "allowed_rows" in a else b
            if "allowed" in a and 0 <= row < len(a["allowed"]):
                index = np.arange(vocabulary)
                x = np.where((a["allowed"][row][index // 32] >> (index % 32).astype(np.uint32)) & 1, x, -np.inf)
            out[b] = x
    return out, size


def _argmax(x):
    """The lowest index of the largest value; NaN and -inf never win, 0 when nothing wins."""
    return np.argmax(np.where(np.isnan(x), -np.inf, x), axis=1)


def _check(got, want, size):
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    assert np.all(np.abs(got[fine].astype(np.float64) - want[fine]) <= HALF_STEP * size[fine])


def _run(gx, logits, a, vocabulary, output="new", tokens=True, fill=None):
    import torch
    batch = logits.shape[0]
    x = dev(logits)
    rules = gx.LogitRules.of(**{k: dev(v) for k, v in a.items()})
    out = {"new": lambda: torch.full(logits.shape, 123.0, device="cuda"), "same": lambda: x, "none": lambda: None}[output]()
    picked = torch.full((batch,), -7, dtype=torch.int32, device="cuda") if tokens else None
    work = torch.full((gx.logit_rules_workspace_bytes(vocabulary, batch),), 0xff, dtype=torch.uint8, device="cuda")
    gx.launch_logit_rules(x, rules, out, picked, work if tokens else None, vocabulary)
    return (None if out is None else host(out)), (None if picked is None else host(picked))


@pytest.mark.parametrize("batch,vocabulary,stride,history,bias,masks", [
    (1, 1, 1, 0, 0, 0), (1, 1, 5, 3, 2, 1), (3, 31, 31, 7, 0, 2), (2, 33, 64, 0, 40, 1), (4, 2048, 2048, 100, 5, 2),
    (4, 2049, 2050, 513, 4095, 3), (7, 5003, 5003, 1, 1, 0), (33, 4096, 4100, 2000, 17, 8), (5, 151936, 151936, 600, 300, 3),
    (2, 248077, 248320, 9000, 100, 2), (300, 700, 701, 20, 3, 300)])
def test_rules_equal_the_formula(device, gx, batch, vocabulary, stride, history, bias, masks):
    rng = np.random.default_rng(vocabulary + batch)
    logits = (rng.standard_normal((batch, stride)) * 3).astype(np.float32)
    a = _problem(rng, batch, vocabulary, history, bias, masks)
    say("rules", batch, vocabulary, stride, history, bias, masks)
    want, size = _formula(logits[:, :vocabulary], a)
    out, tokens = _run(gx, logits, a, vocabulary)
    _check(out[:, :vocabulary], want, size)
    assert np.all(out[:, vocabulary:] == 123.0)
    assert np.array_equal(tokens, _argmax(out[:, :vocabulary]))
    again, only = _run(gx, logits, a, vocabulary, output="same")      # in place, the same bits
    assert np.array_equal(again[:, :vocabulary].view(np.uint32), out[:, :vocabulary].view(np.uint32))
    assert np.array_equal(again[:, vocabulary:], logits[:, vocabulary:]) and np.array_equal(only, tokens)
    assert np.array_equal(_run(gx, logits, a, vocabulary, output="none")[1], tokens)
    assert np.array_equal(_run(gx, logits, a, vocabulary, tokens=False)[0], out)


def test_each_rule_alone(device, gx):
    rng = np.random.default_rng(5)
    batch, vocabulary = 6, 3000
    logits = (rng.standard_normal((batch, vocabulary)) * 3).astype(np.float32)
    a = _problem(rng, batch, vocabulary, 400, 30, 4)
    base = {k: a[k] for k in ("history", "history_lengths")}
    for names in ([], ["repetition"], ["presence"], ["frequency"], ["prompt_lengths", "frequency"],
                  ["prompt_lengths", "repetition", "presence", "frequency"]):
        part = dict(base, **{k: a[k] for k in names}) if names else {}
        say("rules alone", names)
        out, tokens = _run(gx, logits, part, vocabulary)
        _check(out, *_formula(logits, part))
        assert np.array_equal(tokens, _argmax(out))
    for part in ({k: a[k] for k in ("bias_tokens", "bias_values")}, {"allowed": rng.integers(0, 1 << 32, (batch, 94), dtype=np.uint64).astype(np.uint32)}):
        out, tokens = _run(gx, logits, part, vocabulary)
        _check(out, *_formula(logits, part))
        assert np.array_equal(tokens, _argmax(out))


def test_rows_of_a_verify_block_share_a_history(device, gx):
    """Row t of a block sees the committed tokens and the t drafts before it: one list, growing lengths."""
    rng = np.random.default_rng(8)
    batch, vocabulary = 10, 2500
    logits = (rng.standard_normal((batch, vocabulary)) * 3).astype(np.float32)
    a = _problem(rng, batch, vocabulary, 60, rows=2)
    a["history_rows"] = np.repeat([1, 0], 5).astype(np.int32)
    a["history_lengths"] = np.concatenate([np.arange(50, 55), np.arange(30, 35)]).astype(np.uint32)
    a["prompt_lengths"] = np.full(batch, 25, np.uint32)
    say("shared history")
    out, tokens = _run(gx, logits, a, vocabulary)
    _check(out, *_formula(logits, a))
    assert np.array_equal(tokens, _argmax(out))
    a["history_rows"][[0, 7]] = [-1, 2]                               # outside: no history
    _check(_run(gx, logits, a, vocabulary)[0], *_formula(logits, a))


def test_rows_with_nothing_left_and_special_values(device, gx):
    batch, vocabulary = 8, 5000
    rng = np.random.default_rng(9)
    logits = rng.standard_normal((batch, vocabulary)).astype(np.float32)
    logits[0, 17] = np.nan
    logits[1, [40, 4000]] = np.inf
    logits[2] = -np.inf
    logits[3] = np.nan
    logits[4, [2100, 2047, 4999]] = 50.0                              # a tie across slices: the lowest index
    logits[5] = 0.0
    logits[5, ::2] = -0.0
    a = {"allowed": np.full((3, 157), 0xffffffff, np.uint32), "allowed_rows": np.array([0, 0, 0, 0, 0, 0, 1, 2], np.int32)}
    a["allowed"][1] = 0                                               # nothing allowed
    a["allowed"][2] = 0
    a["allowed"][2, 156] = 1 << 7                                     # the last token alone
    a["bias_tokens"] = np.tile(np.array([4999, 3, 4999], np.uint32), (batch, 1))
    a["bias_values"] = np.tile(np.array([7.0, -np.inf, 0.0], np.float32), (batch, 1))
    say("special values")
    out, tokens = _run(gx, logits, a, vocabulary)
    _check(out, *_formula(logits, a))
    assert np.all(out[:3, 3][np.isfinite(logits[:3, 3])] == -np.inf)
    assert list(tokens[1:]) == [40, 0, 0, 2047, 0, 0, 4999]
    assert np.array_equal(tokens, _argmax(out))


def test_long_histories_of_one_token(device, gx):
    """Every count up to the limit of a row, all of one token: no counter runs into its neighbour's bits."""
    vocabulary, length = 100, 524287
    a = {"history": np.full((1, length), 42, np.uint32), "history_lengths": np.array([length], np.uint32),
         "frequency": np.array([0.25], np.float32), "bias_tokens": np.full((1, 4095), 42, np.uint32),
         "bias_values": np.arange(4095, dtype=np.float32)[None]}
    logits = np.ones((1, vocabulary), np.float32)
    say("long history")
    out, tokens = _run(gx, logits, a, vocabulary)
    _check(out, *_formula(logits, a))
    assert out[0, 42] == 1.0 - 0.25 * length + 4094 and tokens[0] == 0
    a["prompt_lengths"] = np.array([length], np.uint32)               # all prompt: seen, not counted
    assert _run(gx, logits, a, vocabulary)[0][0, 42] == 4095.0


def test_rules_in_a_graph_on_another_stream(device, gx):
    import torch
    rng = np.random.default_rng(3)
    batch, vocabulary = 5, 20000
    a = _problem(rng, batch, vocabulary, 300, 20, 5)
    logits = dev((rng.standard_normal((batch, vocabulary)) * 3).astype(np.float32))
    d = {k: dev(v) for k, v in a.items()}
    rules = gx.LogitRules.of(**d)
    out, tokens = empty((batch, vocabulary), np.float32), empty((batch,), np.uint32)
    work = empty((gx.logit_rules_workspace_bytes(vocabulary, batch),), np.uint8)
    say("rules in a graph")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        gx.launch_logit_rules(logits, rules, out, tokens, work)
    for turn in range(4):
        logits.mul_(-1.5)
        d["history_lengths"].add_(1)
        graph.replay()
        got, picked = host(out).copy(), host(tokens).copy()
        a["history_lengths"] = host(d["history_lengths"], np.uint32)
        _check(got, *_formula(host(logits), a))
        assert np.array_equal(picked, _argmax(got))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        eager = torch.zeros_like(out)
        gx.launch_logit_rules(logits, rules, eager, tokens, work, stream=side)
        torch.cuda.synchronize()
        assert np.array_equal(host(eager).view(np.uint32), got.view(np.uint32))


@pytest.mark.parametrize("stride,shift", [(12288, 0), (12289, 0), (12288, 1), (12290, 2)])
def test_unaligned_rows_and_large_batches(device, gx, stride, shift):
    """Rows on 16-byte boundaries or off them, in a batch that takes the larger slices; what lies around a row stays."""
    import torch
    rng = np.random.default_rng(stride + shift)
    batch, vocabulary = 400, 12285
    a = _problem(rng, batch, vocabulary, 70, 9, 30)
    logits = (rng.standard_normal((batch, vocabulary)) * 3).astype(np.float32)
    flat = torch.full((batch * stride + 8,), -9.0, device="cuda")
    out = torch.full((batch * stride + 8,), 123.0, device="cuda")
    view, to = (t[shift:shift + batch * stride].view(batch, stride) for t in (flat, out))
    view[:, :vocabulary] = dev(logits)
    rules = gx.LogitRules.of(**{k: dev(v) for k, v in a.items()})
    tokens = empty((batch,), np.uint32)
    work = empty((gx.logit_rules_workspace_bytes(vocabulary, batch),), np.uint8)
    say("unaligned rows", stride, shift)
    gx.launch_logit_rules(view, rules, to, tokens, work, vocabulary)
    got = host(to)
    _check(got[:, :vocabulary], *_formula(logits, a))
    assert np.all(got[:, vocabulary:] == 123.0) and np.all(host(out)[:shift] == 123.0) and np.all(host(out)[shift + batch * stride:] == 123.0)
    assert np.array_equal(host(tokens), _argmax(got[:, :vocabulary]))


def _formula_fp32(logits, a):
    """The rules in fp32, one rounding an operation, in the order the header gives them."""
    out = logits.copy()
    batch, vocabulary = out.shape
    one = np.float32
    with np.errstate(all="ignore"):
        for b in range(batch):
            x = out[b]
            row = int(a["history_rows"][b]) if "history_rows" in a else b
            if "history" in a and 0 <= row < len(a["history"]):
                tokens = a["history"][row][:a["history_lengths"][b]].astype(np.int64)
                prompt = int(a["prompt_lengths"][b]) if "prompt_lengths" in a else 0
                seen, count = (np.bincount(t[t < vocabulary], minlength=vocabulary) for t in (tokens, tokens[prompt:]))
                factor, f, p = (one(a[k][b]) if k in a else one(d) for k, d in (("repetition", 1), ("frequency", 0), ("presence", 0)))
                x = np.where(seen > 0, np.where(x > 0, x / factor, x * factor), x)
                x = np.where(count > 0, (x - f * count.astype(np.float32)) - p, x)
            if "bias_tokens" in a:
                n = int(a["bias_counts"][b]) if "bias_counts" in a else a["bias_tokens"].shape[1]
                x = x.copy()
                for t, v in {int(t): v for t, v in zip(a["bias_tokens"][b][:n], a["bias_values"][b][:n]) if t < vocabulary}.items():
                    x[t] += v
            row = int(a["allowed_rows"][b]) if "allowed_rows" in a else b
            if "allowed" in a and 0 <= row < len(a["allowed"]):
                index = np.arange(vocabulary)
                x = np.where((a["allowed"][row][index // 32] >> (index % 32).astype(np.uint32)) & 1, x, one(-np.inf))
            assert x.dtype == np.float32
            out[b] = x
    return out


@pytest.mark.parametrize("batch,vocabulary,history,bias,masks", [
    (1, 1, 5, 2, 0), (3, 33, 40, 7, 2), (5, 5003, 700, 300, 3), (33, 4096, 2000, 17, 8), (2, 151936, 9000, 4095, 1), (256, 9001, 300, 30, 0)])
def test_each_operation_is_rounded_once(device, gx, batch, vocabulary, history, bias, masks):
    """The same bits as fp32 operations in the stated order, over small and large magnitudes."""
    rng = np.random.default_rng(vocabulary * 3 + batch)
    logits = (rng.standard_normal((batch, vocabulary)) * 2.0 ** rng.integers(-40, 20, (batch, vocabulary))).astype(np.float32)
    logits[rng.random(logits.shape) < 0.01] = 0
    a = _problem(rng, batch, vocabulary, history, bias, masks)
    say("rules in fp32", batch, vocabulary, history, bias, masks)
    out, tokens = _run(gx, logits, a, vocabulary)
    want = _formula_fp32(logits, a)
    assert np.array_equal(out.view(np.uint32), want.view(np.uint32))
    assert np.array_equal(tokens, _argmax(want))
