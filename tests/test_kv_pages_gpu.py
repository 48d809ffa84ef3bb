"""The paged K/V cache on the GPU against the plain model of kv_pages_model.py: copies, tables and counts are exact,
so every comparison is of whole pools and whole states, bit for bit."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from gpu_util import dev, host, say
from kv_pages_model import PagesModel

pytestmark = pytest.mark.gpu


class Cache:
    """The model and its device twin; every call goes to both."""

    def __init__(self, gx, layers, pages, page_tokens, kv_heads, head_size, sequences, stride, seed=0):
        import torch
        self.gx, self.rng = gx, np.random.default_rng(seed)
        self.model = PagesModel(layers, pages, page_tokens, kv_heads, head_size, sequences, stride, self.rng)
        self.row = (kv_heads, head_size)
        self.k, self.v = (torch.from_numpy(a.copy()).cuda() for a in (self.model.k, self.model.v))
        self.table, self.lengths, self.references = (torch.full(s, 7, dtype=torch.int32, device="cuda")
                                                     for s in ((sequences, stride), (sequences,), (pages,)))
        self.pages = gx.KvPages.of(self.k, self.v, self.table, self.lengths, self.references)
        self.work = torch.full((gx.kv_pages_workspace_bytes(self.pages),), 0x5a, dtype=torch.uint8, device="cuda")
        self.status, self.live = (torch.full((1,), 9, dtype=torch.int32, device="cuda") for _ in range(2))
        gx.launch_kv_pages_reset(self.pages)

    def fork(self, parent, children):
        self.gx.launch_kv_pages_fork(self.pages, parent, children)
        self.model.fork(parent, children)

    def free(self, sequences, keep=None):
        self.gx.launch_kv_pages_free(self.pages, sequences, keep)
        self.model.free(sequences, keep)

    def reserve(self, sequences, tokens):
        self.gx.launch_kv_pages_reserve(self.pages, sequences, tokens, self.status, self.work)
        want = self.model.reserve(sequences, tokens)
        assert int(self.status[0]) == want
        return want

    def append(self, sequences, tokens, layers=None):
        for layer in range(self.k.shape[0]) if layers is None else layers:
            key = self.rng.standard_normal((len(sequences), tokens, *self.row)).astype(np.float16)
            value = self.rng.standard_normal((len(sequences), tokens, *self.row)).astype(np.float32)
            self.gx.launch_kv_pages_append(self.pages, layer, dev(key), dev(value), sequences, tokens)
            self.model.append(layer, key, value, sequences)

    def advance(self, sequences, tokens, counts=None):
        device = None if counts is None else dev(np.array(counts, dtype=np.uint32))
        self.gx.launch_kv_pages_advance(self.pages, sequences, tokens, device)
        self.model.advance(sequences, tokens, counts)

    def grow(self, sequences, tokens):
        assert self.reserve(sequences, tokens) == 0
        self.append(sequences, tokens)
        self.advance(sequences, tokens)

    def compact(self):
        self.gx.launch_kv_pages_compact(self.pages, self.live, self.work)
        assert int(self.live[0]) == self.model.compact()

    def check(self):
        m = self.model
        assert np.array_equal(host(self.lengths), m.lengths)
        assert np.array_equal(host(self.table), m.table_array())
        assert np.array_equal(host(self.references), m.references)
        assert np.array_equal(host(self.k).view(np.uint16), m.k.view(np.uint16))
        assert np.array_equal(host(self.v).view(np.uint16), m.v.view(np.uint16))


@pytest.mark.parametrize("page_tokens,kv_heads,head_size", [(16, 2, 128), (32, 1, 256), (64, 8, 128), (128, 4, 256)])
def test_fork_reserve_append_free_compact(device, gx, page_tokens, kv_heads, head_size):
    say("pages", page_tokens, kv_heads, head_size)
    c = Cache(gx, 2, 40, page_tokens, kv_heads, head_size, 8, 12, seed=page_tokens)
    c.check()
    c.grow([3], 2 * page_tokens + 5)
    c.fork(3, [0, 1, 5])
    c.check()
    c.grow([0, 1], 1)          # both copy the tail, 3 and 5 still share it
    c.check()
    c.grow([5, 3], 3)          # the last two holders: 5 copies, 3 keeps the page
    c.check()
    c.fork(1, [2, 5])          # 5 gives its pages back first
    c.grow([2, 0, 5, 1, 3], page_tokens)
    c.check()
    c.free([3, 0], [page_tokens + 1, 0])
    c.check()
    c.compact()
    c.check()
    c.grow([3], 1)             # cut inside a page that others hold: copied
    c.grow([4], 3 * page_tokens)
    c.check()
    c.free([1, 2, 3, 4, 5])
    c.compact()
    c.check()
    assert host(c.references).sum() == 0


@pytest.mark.parametrize("seed", range(6))
def test_random_calls_equal_the_model(device, gx, seed):
    rng = np.random.default_rng(100 + seed)
    page = int(rng.choice([16, 32]))
    c = Cache(gx, int(rng.integers(1, 4)), int(rng.integers(20, 60)), page, 1, 128, 7, int(rng.integers(3, 9)), seed)
    say("random calls", seed)
    for step in range(60):
        pick = lambda: [int(i) for i in rng.permutation(7)[:rng.integers(1, 6)]]  # noqa: E731
        what = rng.choice(["grow", "grow", "grow", "fork", "free", "cut", "compact", "advance"])
        if what == "grow":
            who, n = pick(), int(rng.integers(1, page + 10))
            if c.reserve(who, n) == 0:
                c.append(who, n)
                c.advance(who, n, [int(rng.integers(0, n + 3)) for _ in who] if rng.random() < 0.4 else None)
        elif what == "fork":
            who = pick()
            c.fork(who[0], who[1:] or [(who[0] + 1) % 7])
        elif what == "free":
            c.free(pick()[:2])
        elif what == "cut":
            who = pick()
            c.free(who, [int(rng.integers(0, 3 * page)) for _ in who])
        elif what == "compact":
            c.compact()
        else:                  # rows past the reserved pages are skipped
            who = pick()
            c.append(who, page + 3, layers=[0])
        if step % 10 == 9:
            c.check()
    c.check()


def test_a_pool_that_is_too_small_changes_nothing(device, gx):
    c = Cache(gx, 1, 10, 16, 1, 128, 4, 20)
    c.grow([0], 16 * 6 + 1)
    c.fork(0, [1, 2])
    say("pool too small")
    assert c.reserve([1, 2], 17) == 1    # 2 copies + 2 new pages, 3 left
    c.check()
    assert c.reserve([1, 2], 1) == 0     # 2 copies
    c.check()
    assert c.reserve([0], 16 * 20) == 1  # past the table row
    c.check()


def test_many_pages_take_more_than_one_round(device, gx):
    """More pages than one pass of the planning workgroup covers, and more new pages than one window of ranks."""
    pages = 70001
    c = Cache(gx, 1, pages, 16, 1, 128, 3, 68000)
    say("many pages")
    c.grow([0], 16 * 33000 - 3)
    c.grow([1], 16 * 300 + 1)
    c.fork(1, [2])
    c.free([0])
    assert c.reserve([2], 16 * 34000) == 0
    c.check()
    c.compact()
    c.check()
    c.free([1])
    c.compact()
    c.check()


def test_listed_calls_at_their_limit(device, gx):
    """512 sequences in one call, all holding one tail page, one of them not in the list."""
    c = Cache(gx, 1, 600, 16, 1, 128, 513, 2)
    c.grow([512], 5)
    say("512 sequences")
    c.fork(512, list(range(512)))
    c.grow(list(range(512)), 1)
    c.check()
    c.free(list(range(512)), [5] * 512)
    c.fork(0, [512])
    c.check()


def test_append_leaves_shared_pages_alone(device, gx):
    """Rows for a page that another sequence holds are skipped until a reserve has made it private."""
    c = Cache(gx, 1, 12, 16, 1, 128, 4, 4)
    c.grow([0], 21)
    c.fork(0, [1, 2])
    c.free([1], [18])
    say("append to shared pages")
    c.append([0, 1, 2], 20)
    c.check()
    assert c.reserve([1], 2) == 0
    c.append([0, 1, 2], 20)
    c.check()
    assert c.reserve([2, 0], 20) == 0
    c.append([0, 1, 2], 20)
    c.check()


def test_copy_pages(device, gx):
    c = Cache(gx, 3, 12, 64, 2, 128, 2, 4)
    say("copy pages")
    gx.launch_kv_pages_copy(c.pages, [0, 0, 11], [5, 7, 6])
    c.model.copy([0, 0, 11], [5, 7, 6])
    c.check()


def test_default_list_is_the_first_sequences(device, gx):
    c = Cache(gx, 1, 12, 16, 1, 128, 4, 2)
    say("default list")
    gx.check(gx.lib().gfxinfer_launch_kv_pages_reserve(ctypes.byref(c.pages), None, 3, 4, c.status.data_ptr(), c.work.data_ptr(),
                                                       c.work.numel(), None))
    c.model.reserve([0, 1, 2], 4)
    gx.check(gx.lib().gfxinfer_launch_kv_pages_advance(ctypes.byref(c.pages), None, 3, 4, None, None))
    c.model.advance([0, 1, 2], 4)
    c.check()


def test_damaged_table_entries_are_not_followed(device, gx):
    """Entries outside the pool read as missing: nothing is copied, written or counted for them."""
    c = Cache(gx, 1, 8, 16, 1, 128, 3, 4)
    c.grow([0], 20)
    c.grow([2], 16)
    say("damaged table")
    c.table[0, 1] = 1000
    c.table[1, 0] = -5
    before = [host(t).copy() for t in (c.k, c.v)]
    gx.launch_kv_pages_append(c.pages, 0, dev(np.ones((1, 4, 1, 128), np.float16)), dev(np.ones((1, 4, 1, 128), np.float32)), [0], 4)
    gx.launch_kv_pages_reserve(c.pages, [0], 2, c.status, c.work)
    gx.launch_kv_pages_free(c.pages, [0, 1])
    gx.launch_kv_pages_compact(c.pages, c.live, c.work)
    assert int(c.live[0]) == 2          # page 1 is still counted for the entry that was lost, and page 2 is used
    assert np.array_equal(host(c.references)[:3], [1, 1, 0])
    assert np.array_equal(host(c.table), [[-1] * 4, [-1] * 4, [0, -1, -1, -1]])
    assert np.array_equal(before[0][:, 1], host(c.k)[:, 1]) and np.array_equal(before[0][:, 2], host(c.k)[:, 0])


def test_graph_replays_and_other_stream(device, gx):
    """A captured fork + reserve + append + advance, replayed with other work between, equals the model each time."""
    import torch
    c = Cache(gx, 2, 64, 16, 1, 128, 6, 8, seed=3)
    c.grow([0], 21)
    keys, values = ([dev(c.rng.standard_normal((3, 2, 1, 128)).astype(t)) for _ in range(2)]
                    for t in (np.float16, np.float32))

    def step(stream=None):
        gx.launch_kv_pages_fork(c.pages, 0, [1, 2, 3], stream=stream)
        gx.launch_kv_pages_reserve(c.pages, [1, 2, 3], 2, c.status, c.work, stream=stream)
        for layer in range(2):
            gx.launch_kv_pages_append(c.pages, layer, keys[layer], values[layer], [1, 2, 3], 2, stream=stream)
        gx.launch_kv_pages_advance(c.pages, [1, 2, 3], 2, stream=stream)

    def model_step():
        c.model.fork(0, [1, 2, 3])
        assert c.model.reserve([1, 2, 3], 2) == 0
        for layer in range(2):
            c.model.append(layer, host(keys[layer]), host(values[layer]), [1, 2, 3])
        c.model.advance([1, 2, 3], 2)

    say("other stream")
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    step(other)
    torch.cuda.current_stream().wait_stream(other)
    model_step()
    c.check()
    say("graph capture")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    for turn in range(4):
        c.grow([0], 5 + 7 * turn)
        c.grow([2], 3)
        if turn == 2:
            c.free([0], [17])
            c.compact()
        graph.replay()
        model_step()
        c.check()


def test_operands_in_host_memory(device, gx):
    """Pinned memory is read and written like the GPU's; other host memory is refused before anything is launched."""
    import torch
    c = Cache(gx, 1, 8, 16, 1, 128, 2, 4)
    say("host memory")
    c.status = torch.full((1,), 9, dtype=torch.int32, pin_memory=True)
    gx.launch_kv_pages_reserve(c.pages, [0], 5, c.status, c.work)
    torch.cuda.synchronize()
    assert int(c.status[0]) == c.model.reserve([0], 5) == 0
    key, value = torch.zeros(1, 5, 1, 128, dtype=torch.float16), torch.zeros(1, 5, 1, 128)
    for k, v in ((key, value.cuda()), (key.cuda(), value)):
        with pytest.raises(ValueError, match="memory"):
            gx.launch_kv_pages_append(c.pages, 0, k, v, [0], 5)
    with pytest.raises(ValueError, match="key"):
        gx.launch_kv_pages_append(c.pages, 0, key.cuda(), value.cuda(), [0, 1], 5)
    c.check()


@pytest.mark.parametrize("order", [[0, 1], [1, 0], [0], [1]])
@pytest.mark.parametrize("commit", [True, False])
def test_rows_appended_before_a_fork(device, gx, commit, order):
    """A parent's rows past its length: committed before the next reserve they are kept whoever copies the tail page; if not,
    the parent's copy holds the committed rows, and the appended ones are appended again."""
    c = Cache(gx, 2, 12, 16, 1, 128, 3, 4)
    c.grow([0], 20)
    assert c.reserve([0], 5) == 0
    c.append([0], 5)
    appended = [c.model.rows(layer, 0, 25) for layer in range(2)]
    say("rows before a fork", commit, order)
    c.fork(0, [1])
    c.check()
    if commit:
        c.advance([0], 5)
    assert c.reserve(order, 4) == 0
    c.check()
    if not commit:
        assert c.reserve([0], 5) == 0
        for layer, (k, v) in enumerate(appended):
            rows = [x[None, 20:] for x in (k.astype(np.float16), v.astype(np.float32))]
            gx.launch_kv_pages_append(c.pages, layer, *(dev(x) for x in rows), [0], 5)
            c.model.append(layer, *rows, [0])
        c.advance([0], 5)
    c.check()
    for layer, (k, v) in enumerate(appended):
        got = c.model.rows(layer, 0, 25)
        assert np.array_equal(got[0], k) and np.array_equal(got[1], v)
    c.grow([1], 9)
    c.check()


def test_a_recorded_step_whose_reserve_fails(device, gx):
    """Counts taken from the status: replays after the pool is full change nothing, and the step goes on once pages are free."""
    import torch
    c = Cache(gx, 1, 5, 16, 1, 128, 3, 5, seed=4)
    c.grow([0, 1], 20)                                        # four of five pages
    key, value = dev(c.rng.standard_normal((2, 10, 1, 128)).astype(np.float16)), dev(c.rng.standard_normal((2, 10, 1, 128)).astype(np.float32))
    counts = torch.zeros(2, dtype=torch.int32, device="cuda")
    c.status.zero_()
    say("recorded step")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        gx.launch_kv_pages_reserve(c.pages, [0, 1], 10, c.status, c.work)
        gx.launch_kv_pages_append(c.pages, 0, key, value, [0, 1], 10)
        counts.copy_((c.status == 0).to(torch.int32).mul(10).expand(2))
        gx.launch_kv_pages_advance(c.pages, [0, 1], 10, counts)
    for want in (0, 1, 1, 0, 1):                              # 20 -> 30 inside the pages; then two pages, one left
        if want == 0 and c.model.lengths[0] == 30:
            c.free([1], [10])
        graph.replay()
        assert int(c.status[0]) == want == c.model.reserve([0, 1], 10)
        c.model.append(0, host(key), host(value), [0, 1])
        if want == 0:
            c.model.advance([0, 1], 10)
        c.check()
