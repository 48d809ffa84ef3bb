"""Products in 8-bit integers, chunk attention, received weights and eviction together, as a server of several conversations
uses them within a budget: prompts in ragged chunks, then steps of a token each.  Two layers around a random input; every
operator is checked on what the one before it gave: codes, products, the cache and the evictions bit for bit, attention and
weights in 64 bits with the tolerances of their own tests.  Then the decoding step recorded once and replayed."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import dev, host, say
from test_kv_chunks_gpu import Chunks, _check_weights
from test_kv_evict_gpu import Bounded, Cache, gx_bytes
from test_w8a8_gpu import _codes_of, _want

pytestmark = pytest.mark.gpu
LAYERS, HIDDEN = 2, 320


class Server:
    def __init__(self, gx, heads, page, sequences, budget, first, recent, seed):
        import torch
        self.gx, self.torch, self.heads = gx, torch, heads
        self.budget, self.first, self.recent = budget, first, recent
        q_heads, kv_heads, d = heads
        rng = self.rng = np.random.default_rng(seed)
        stride = -(-(budget + 40) // page)
        self.model = Bounded(LAYERS, sequences * stride + 3, page, kv_heads, d, sequences + 1, stride, rng)
        self.cache = Cache(gx, self.model)
        # [out][in] codes and a scale for each output: queries, keys, values and the way back, for each layer.
        sizes = {"q": (q_heads * d, HIDDEN), "k": (kv_heads * d, HIDDEN), "v": (kv_heads * d, HIDDEN), "o": (HIDDEN, q_heads * d)}
        self.host_weights = [{n: (rng.integers(-127, 128, s, dtype=np.int8), (rng.random(s[0]) * 0.5 + 0.5).astype(np.float32) / np.float32(73 * s[1] ** 0.5))
                              for n, s in sizes.items()} for _ in range(LAYERS)]
        self.weights = [{n: (dev(w), dev(s)) for n, (w, s) in layer.items()} for layer in self.host_weights]
        self.work = {}

    def scratch(self, name, size):
        """A workspace each: steps of other sizes do not share one that a recorded step keeps."""
        if name not in self.work or self.work[name].numel() < size:
            self.work[name] = self.torch.full((max(16, size),), 0xff, dtype=self.torch.uint8, device="cuda")
        return self.work[name]

    def product(self, layer, name, x, out):
        codes = self.torch.empty(x.shape, dtype=self.torch.int8, device="cuda")
        scales = self.torch.empty(x.shape[0], device="cuda")
        self.gx.launch_quantize_rows_i8(x, codes, scales)
        w, s = self.weights[layer][name]
        self.gx.launch_w8a8_gemm(w, s, codes, scales, out, self.scratch("product", self.gx.w8a8_gemm_workspace_bytes(*w.shape, x.shape[0])))
        return codes, scales

    def step(self, x, tokens, seen=None):
        """Rows x [sum(tokens), HIDDEN] through both layers; seen: called with what each operator took and gave."""
        gx, torch, cache = self.gx, self.torch, self.cache
        q_heads, kv_heads, d = self.heads
        n, rows, listed = len(tokens), sum(tokens), list(range(len(tokens)))
        seen = seen or (lambda *a: None)
        state = self.scratch("pages", gx.kv_pages_workspace_bytes(cache.pages))
        for t in sorted(set(tokens)):                          # reserve and append take one length at a time
            gx.launch_kv_pages_reserve(cache.pages, [i for i in listed if tokens[i] == t], t, cache.status, state)
        gx.launch_kv_weights_begin(cache.pages, cache.weights, listed, tokens)
        seen("begin", tokens)
        for layer in range(LAYERS):
            half = lambda size: torch.empty((rows, size), dtype=torch.float16, device="cuda")  # noqa: E731
            query, key, value, out, back = half(q_heads * d), half(kv_heads * d), torch.empty((rows, kv_heads * d), device="cuda"), half(q_heads * d), half(HIDDEN)
            for name, y in (("q", query), ("k", key), ("v", value)):
                seen("product", layer, name, x, *self.product(layer, name, x, y), y)
            at = 0
            for i, t in enumerate(tokens):
                gx.launch_kv_pages_append(cache.pages, layer, key[at:at + t], value[at:at + t], [i], t)
                at += t
            seen("append", layer, key, value, tokens)
            sums = torch.empty((rows, q_heads), device="cuda")
            gx.launch_kv_pages_chunk_attention(cache.pages, layer, query, None, out, sums, listed, tokens, q_heads,
                                               self.scratch("attention", gx.kv_pages_chunk_attention_workspace_bytes(cache.pages, tokens, q_heads)))
            seen("attention", layer, query, out, sums, tokens)
            gx.launch_kv_weights_add(cache.pages, cache.weights, layer, query, sums, listed, tokens, q_heads,
                                     self.scratch("weights", gx.kv_weights_workspace_bytes(cache.pages, tokens, q_heads)))
            seen("weights", layer, query, sums, tokens)
            seen("product", layer, "o", out, *self.product(layer, "o", out, back), back)
            x = back
        for t in sorted(set(tokens)):
            gx.launch_kv_pages_advance(cache.pages, [i for i in listed if tokens[i] == t], t)
        gx.launch_kv_pages_evict(cache.pages, cache.weights, listed, self.budget, self.first, self.recent, cache.status,
                                 self.scratch("evict", gx_bytes(gx, cache.pages, n, self.budget)))
        seen("evict", tokens)
        return x

    # ---- the checks ------------------------------------------------------------------------

    def chunks(self, layer, query, tokens):
        """The rows of the model's cache as the attention's own tests describe them."""
        m, c = self.model, Chunks.__new__(Chunks)
        c.heads, c.page, c.lengths, c.tokens, c.gate = self.heads, m.page, m.lengths[:len(tokens)], list(tokens), None
        c.hidden = [np.zeros(n + t, bool) for n, t in zip(c.lengths, tokens)]
        c.rows = []
        for i, n in enumerate(c.lengths):
            j = np.arange(n + tokens[i])
            page = np.array(m.table[i], np.int64)[j // m.page]
            c.rows.append([pool[layer, page, j % m.page] for pool in (m.k, m.v)])
        c.query = host(query).reshape(-1, self.heads[0], self.heads[2])
        return c

    def see(self, what, *a):
        m = self.model
        if what == "begin":
            for t in sorted(set(a[0])):
                assert m.reserve([i for i in range(len(a[0])) if a[0][i] == t], t) == 0
            m.begin(range(len(a[0])), a[0])
            self.cache.check()
            self.before = m.weight.copy()
        elif what == "product":
            layer, name, x, codes, scales, y = a
            want, wanted = _codes_of(host(x.float()))
            assert np.array_equal(host(codes), want) and np.array_equal(host(scales), wanted)
            w, s = self.host_weights[layer][name]
            got = host(y)
            assert np.array_equal(got, _want(w, s, want, wanted, got.dtype == np.float16))
        elif what == "append":
            layer, key, value, tokens = a
            rows, at = (-1, self.heads[1], self.heads[2]), 0
            k, v = host(key).reshape(rows), host(value).reshape(rows)
            for i, t in enumerate(tokens):
                m.append(layer, k[None, at:at + t], v[None, at:at + t], [i])
                at += t
        elif what == "attention":
            layer, query, out, sums, tokens = a
            self.chunks(layer, query, tokens).check(host(out).reshape(-1, self.heads[0], self.heads[2]), host(sums))
        elif what == "weights":
            layer, query, sums, tokens = a
            got = host(self.cache.weight)
            _check_weights(self.chunks(layer, query, tokens), got, host(sums), self.before)
            self.before = m.weight[:] = got
        else:
            for i, t in enumerate(a[0]):
                m.advance([i], t)
            assert m.evict(range(len(a[0])), self.budget, self.first, self.recent) == 0
            self.cache.check()

    def input(self, rows):
        return dev(self.rng.standard_normal((rows, HIDDEN)).astype(np.float16))


@pytest.mark.parametrize("heads,page", [((4, 2, 128), 16), ((6, 1, 256), 32), ((40, 8, 128), 64)])
def test_conversations_within_a_budget(device, gx, heads, page):
    import torch
    s = Server(gx, heads, page, 3, 70, 4, 20, page)
    for tokens in ([33, 1, 17], [40, 9, 40], [1, 40, 2], [1, 1, 1], [1, 1, 1]):
        say("a step of", tokens, heads, page)
        out = s.step(s.input(sum(tokens)), tokens, s.see)
        assert bool(torch.isfinite(out).all())
    assert max(s.model.dropped) > 0 and max(s.model.lengths) == 70


@pytest.mark.parametrize("heads,page", [((4, 2, 128), 16), ((6, 1, 256), 32)])
def test_a_recorded_step(device, gx, heads, page):
    """The same inputs through a recorded step and through eager calls on a cache of its own: the same bits, again and again."""
    import torch
    eager, recorded = (Server(gx, heads, page, 3, 70, 4, 20, 7) for _ in range(2))
    x = eager.input(100)
    for s in (eager, recorded):
        for rows in ([60, 5, 35], [40, 30, 30]):
            s.step(x, rows)
    static, tokens = eager.input(3), [1, 1, 1]
    recorded.step(static, tokens)                              # the workspaces of a step of this size
    eager.step(static, tokens)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = recorded.step(static, tokens)
    say("recorded steps", heads, page)
    for _ in range(4):
        static.copy_(eager.input(3))
        graph.replay()
        want = eager.step(static.clone(), tokens)
        torch.cuda.synchronize()
        assert np.array_equal(host(out).view(np.int16), host(want).view(np.int16))
        for name in ("k", "v", "table", "lengths", "references", "weight", "position", "dropped"):
            a, b = (host(getattr(s.cache, name)) for s in (eager, recorded))
            assert np.array_equal(a.view(np.int16), b.view(np.int16)), name
