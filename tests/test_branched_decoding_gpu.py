"""The paged cache, the attention over it and the logit rules together, as a sampler of several continuations uses them:
one prompt, its sequence forked, then steps of reserve, append, attention, logits with rules, advance.  The model around
them is a table lookup (a token's query, key and value rows) and one product, so every step can be checked against the
definitions: the whole cache against the plain model bit for bit, the attention and the logits in 64 bits with the
tolerances of their own tests, the tokens exactly."""
from __future__ import annotations

import math

import numpy as np
import pytest

from gpu_util import dev, empty, host, say
from kv_pages_model import PagesModel
from test_logit_rules_gpu import _argmax, _check, _formula

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


class Branches:
    """Slot 0 the prompt, slots 1..n the branches; the device side and the plain model of everything."""

    def __init__(self, gx, heads, page, n, vocabulary, seed):
        import torch
        self.gx, self.n, self.vocabulary, self.heads = gx, n, vocabulary, heads
        q_heads, kv_heads, d = heads
        rng = self.rng = np.random.default_rng(seed)
        self.model = PagesModel(1, 64, page, kv_heads, d, n + 1, 12, rng)
        self.k, self.v = dev(self.model.k), dev(self.model.v)
        self.table, self.lengths, self.references = empty((n + 1, 12), np.int32), empty((n + 1,), np.int32), empty((64,), np.int32)
        self.pages = gx.KvPages.of(self.k, self.v, self.table, self.lengths, self.references)
        self.pages_work = empty((gx.kv_pages_workspace_bytes(self.pages),), np.uint8)
        self.status = empty((1,), np.int32)
        gx.launch_kv_pages_reset(self.pages)
        normal = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        # Rows of every token; the output product is small enough that logits stay apart by more than its rounding.
        self.rows = {"q": normal(vocabulary, q_heads, d).astype(np.float16), "k": normal(vocabulary, kv_heads, d).astype(np.float16),
                     "v": normal(vocabulary, kv_heads, d), "gate": normal(vocabulary, q_heads, 2 * d)}
        self.device_rows = {k: dev(x) for k, x in self.rows.items()}
        self.head = dev(normal(q_heads * d, vocabulary))
        self.shared = 0
        self.torch = torch

    def prompt(self, tokens, block):
        """Blocks of the prompt through reserve, append and advance of slot 0."""
        for i in range(0, len(tokens), block):
            part = np.array(tokens[i:i + block])
            self.gx.launch_kv_pages_reserve(self.pages, [0], len(part), self.status, self.pages_work)
            self.gx.launch_kv_pages_append(self.pages, 0, dev(self.rows["k"][part]), dev(self.rows["v"][part]), [0], len(part))
            self.gx.launch_kv_pages_advance(self.pages, [0], len(part))
            assert int(self.status[0]) == 0 and self.model.reserve([0], len(part)) == 0
            self.model.append(0, self.rows["k"][part][None], self.rows["v"][part][None], [0])
            self.model.advance([0], len(part))
        self.shared = len(tokens)
        self.gx.launch_kv_pages_fork(self.pages, 0, range(1, self.n + 1))
        self.model.fork(0, list(range(1, self.n + 1)))

    def check_cache(self):
        m = self.model
        assert np.array_equal(host(self.lengths), m.lengths) and np.array_equal(host(self.table), m.table_array())
        assert np.array_equal(host(self.references), m.references)
        assert np.array_equal(host(self.k).view(np.uint16), m.k.view(np.uint16))
        assert np.array_equal(host(self.v).view(np.uint16), m.v.view(np.uint16))

    def buffers(self, block, rules):
        q_heads, _, d = self.heads
        t = self.torch
        self.block, self.rules = block, self.gx.LogitRules.of(**rules)
        self.output = t.zeros((self.n, block, q_heads, d), dtype=t.float16, device="cuda")
        self.attention_work = empty((self.gx.kv_pages_attention_workspace_bytes(self.pages, self.n, block, q_heads, self.shared),), np.uint8)
        self.logits = t.zeros((self.n * block, self.vocabulary), device="cuda")
        self.ruled = t.zeros_like(self.logits)
        self.picked = t.zeros(self.n * block, dtype=t.int32, device="cuda")
        self.rules_work = empty((self.gx.logit_rules_workspace_bytes(self.vocabulary, self.n * block),), np.uint8)

    def device_step(self, tokens):
        """tokens: device int64 [n, block], the last picked ones; everything by launches and torch indexing."""
        gx, who = self.gx, range(1, self.n + 1)
        rows = {k: x[tokens] for k, x in self.device_rows.items()}
        gx.launch_kv_pages_reserve(self.pages, who, self.block, self.status, self.pages_work)
        gx.launch_kv_pages_append(self.pages, 0, rows["k"], rows["v"], who, self.block)
        gx.launch_kv_pages_gated_attention(self.pages, 0, rows["q"], rows["gate"], self.output, who, self.block, self.heads[0],
                                           self.shared, self.attention_work)
        self.torch.matmul(self.output.view(self.n * self.block, -1).float(), self.head, out=self.logits)
        gx.launch_logit_rules(self.logits, self.rules, self.ruled, self.picked, self.rules_work)

    def check_step(self, tokens, rules):
        """The same step on the plain model, then every output of the device's."""
        who = list(range(1, self.n + 1))
        tokens = np.asarray(tokens)
        assert int(self.status[0]) == 0 and self.model.reserve(who, self.block) == 0
        self.model.append(0, self.rows["k"][tokens], self.rows["v"][tokens], who)
        q_heads, kv_heads, d = self.heads
        got = host(self.output).astype(np.float64)
        for i, s in enumerate(who):
            for t in range(self.block):
                n = self.model.lengths[s] + t + 1
                k, v = self.model.rows(0, s, n)
                for h in range(q_heads):
                    q, kk, vv = self.rows["q"][tokens[i, t], h].astype(np.float64), k[:, h * kv_heads // q_heads], v[:, h * kv_heads // q_heads]
                    score = kk @ q / math.sqrt(d)
                    w = np.exp(score - score.max())
                    w /= w.sum()
                    g = 1 / (1 + np.exp(-self.rows["gate"][tokens[i, t], h, d:].astype(np.float64)))
                    want = w @ vv * g
                    # The tolerance of the attention's own test.
                    e = 2 * (d + 8) * U * (np.abs(kk) @ np.abs(q)).max() / math.sqrt(d) + 2.0 ** -21
                    tol = (2 * e + (n / 2 + 64) * U) * (w @ np.abs(vv)) * g + np.maximum(np.abs(want) * 2.0 ** -11, 2.0 ** -25) * (1 + 2.0 ** -10)
                    assert np.all(np.abs(got[i, t, h] - want) <= tol)
        ruled = host(self.ruled)
        _check(ruled, *_formula(host(self.logits), rules))
        assert np.array_equal(host(self.picked), _argmax(ruled))


@pytest.mark.parametrize("heads,page", [((10, 2, 128), 16), ((6, 1, 256), 32)])
def test_branches_of_one_prompt(device, gx, heads, page):
    """Four branches with their own penalties, biases and grammar, one token a step, captured after the first step."""
    import torch
    n, vocabulary = 4, 700
    b = Branches(gx, heads, page, n, vocabulary, seed=page)
    prompt = [int(x) for x in b.rng.integers(0, vocabulary, 2 * page + 5)]
    say("branches", heads, page)
    b.prompt(prompt, 32)
    b.check_cache()
    history = empty((n, 100), np.int32)
    history[:, :len(prompt)] = dev(np.array(prompt, np.int32))
    rules = {"history": history, "history_lengths": torch.full((n,), len(prompt), dtype=torch.int32, device="cuda"),
             "prompt_lengths": torch.full((n,), len(prompt), dtype=torch.int32, device="cuda"),
             "repetition": dev(np.array([1.0, 1.2, 1.0, 1.5], np.float32)), "presence": dev(np.array([0, 0.5, 40, 0], np.float32)),
             "frequency": dev(np.array([0, 0.1, 0.2, 30], np.float32)),
             "allowed": dev(b.rng.integers(0, 1 << 32, (2, 22), dtype=np.uint64).astype(np.uint32)),
             "allowed_rows": dev(np.array([-1, 0, 1, -1], np.int32))}
    b.buffers(1, rules)
    tokens = torch.full((n, 1), prompt[-1], dtype=torch.int64, device="cuda")
    step = torch.zeros(1, dtype=torch.int64, device="cuda")

    def whole():
        b.device_step(tokens)
        gx.launch_kv_pages_advance(b.pages, range(1, n + 1), 1)
        tokens.copy_(b.picked.view(n, 1))
        rules["history"].scatter_(1, rules["history_lengths"].long().view(n, 1), b.picked.view(n, 1))
        rules["history_lengths"].add_(1)
        step.add_(1)

    graph, seen = torch.cuda.CUDAGraph(), set()
    for turn in range(9):
        before = {k: host(x).copy() for k, x in rules.items()}
        for k in ("history", "history_lengths", "prompt_lengths", "allowed"):
            before[k] = before[k].view(np.uint32)
        given = host(tokens).copy()
        if turn == 1:
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                whole()
        if turn == 0:
            whole()
        else:
            graph.replay()
        b.check_step(given, before)
        b.model.advance(list(range(1, n + 1)), 1)
        b.check_cache()
        picked = host(b.picked)
        seen.update(int(x) for x in picked)
    assert int(step[0]) == 9 and len(seen) > 9
    assert len({tuple(row) for row in host(history)[:, len(prompt):len(prompt) + 9].tolist()}) > 1


def test_verify_blocks_accept_and_fork_again(device, gx):
    """Blocks of four drafts a branch, accepted counts from the device; then the best branch replaces the others."""
    import torch
    n, block, vocabulary, heads = 3, 4, 500, (8, 2, 128)
    b = Branches(gx, heads, 16, n, vocabulary, seed=9)
    prompt = [int(x) for x in b.rng.integers(0, vocabulary, 30)]
    say("verify blocks")
    b.prompt(prompt, 7)
    who = list(range(1, n + 1))
    for turn in range(4):
        drafts = b.rng.integers(0, vocabulary, (n, block)).astype(np.int64)
        # Row t of a block sees the committed tokens (here: the prompt) and the drafts up to its own.
        lists = np.concatenate([np.tile(np.array(prompt, np.uint32), (n, 1)), drafts.astype(np.uint32)], 1)
        rules = {"history": dev(lists), "history_rows": dev(np.repeat(np.arange(n), block).astype(np.int32)),
                 "history_lengths": dev(np.tile(len(prompt) + 1 + np.arange(block), n).astype(np.uint32)),
                 "prompt_lengths": dev(np.full(n * block, len(prompt), np.uint32)),
                 "repetition": dev(np.full(n * block, 1.3, np.float32)), "frequency": dev(np.full(n * block, 2.0, np.float32))}
        b.buffers(block, rules)
        b.device_step(dev(drafts))
        b.check_step(drafts, {"history": lists, "history_rows": np.repeat(np.arange(n), block), "history_lengths": host(rules["history_lengths"], np.uint32),
                              "prompt_lengths": host(rules["prompt_lengths"], np.uint32), "repetition": host(rules["repetition"]), "frequency": host(rules["frequency"])})
        accepted = b.rng.integers(0, block + 1, n).astype(np.uint32)
        gx.launch_kv_pages_advance(b.pages, who, block, dev(accepted))
        b.model.advance(who, block, [int(x) for x in accepted])
        b.check_cache()
        if turn == 1:                                        # branch 2 wins: the others become copies of it
            gx.launch_kv_pages_fork(b.pages, 2, [1, 3])
            b.model.fork(2, [1, 3])
            gx.launch_kv_pages_free(b.pages, [0])
            b.model.free([0])
            b.shared = b.model.lengths[2]
            live = empty((1,), np.int32)
            gx.launch_kv_pages_compact(b.pages, live, b.pages_work)
            assert int(live[0]) == b.model.compact()
            b.check_cache()
