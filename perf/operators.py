"""Operators of branched decoding, as cases that can be timed and checked: many continuations of one prompt.

`attention`: gated GQA attention over K/V pages for a batch whose sequences share a prefix.
`branch`: one step of a sampler's cache: children forked from a parent, their tail pages made private, a block of
tokens appended in every layer.  `churn`: a sequence ends, the pool is compacted, another one is admitted.
`rules`: penalties, biases and grammar masks on the logits, with the greedy token.

With `own` false the plain form runs, elementary torch operations in 32 bits; with `own` true the calls of
gfxinfer_amd.  `exact` states each operator once more, in 64 bits, sequence by sequence.
"""
import math

import torch

own = False

DEVICE = "cuda"
HEADS = {"27b": (40, 8, 128), "reference": (24, 4, 256)}   # query heads, KV heads, head size
LAYERS = 16                                                # full-attention layers of both shapes


def listed():
    return [
        # Four continuations of a short prompt, one token each: a decode step where latency counts.
        dict(name="attention_4_short", op="attention", shape="27b", count=4, tokens=1, shared=512, own_min=1, own_max=48,
             page=16),
        # A sampler's ordinary step: 32 continuations some hundred tokens into their answers.
        dict(name="attention_32_sampling", op="attention", shape="27b", count=32, tokens=1, shared=4096, own_min=32,
             own_max=480, page=64),
        # Verify blocks of depth 4 for eight branches whose prefix ends inside a page.
        dict(name="attention_8_verify", op="attention", shape="reference", count=8, tokens=5, shared=2000, own_min=1,
             own_max=200, page=32),
        # 16 independent conversations (nothing shared) of very different lengths, 256-wide heads.
        dict(name="attention_16_ragged", op="attention", shape="reference", count=16, tokens=1, shared=0, own_min=1,
             own_max=4090, page=16),
        # 64 continuations of a long document.
        dict(name="attention_64_long", op="attention", shape="27b", count=64, tokens=1, shared=32768, own_min=100,
             own_max=900, page=128),
        # Three children of a chat prompt, one token each.
        dict(name="branch_3", op="branch", shape="27b", layers=LAYERS, page=16, parent=509, children=3, tokens=1,
             others=40),
        # 63 children late in a conversation, verify blocks of five tokens.
        dict(name="branch_63", op="branch", shape="27b", layers=LAYERS, page=64, parent=3900, children=63, tokens=5,
             others=100),
        # A short request leaves and another comes, twice.
        dict(name="churn_short", op="churn", shape="27b", layers=LAYERS, page=16, length=77, others=20),
        # Long prompts leave and come.
        dict(name="churn_long", op="churn", shape="reference", layers=LAYERS, page=64, length=2000, others=60),
        # A five-token verify block under a grammar.
        dict(name="rules_5_grammar", op="rules", batch=5, rows=151936, vocabulary=151936, history=600, prompt=509,
             bias=0, masked=True, penalties=True),
        # Ordinary sampling step, long histories, biases, no grammar; rows wider than the tokenizer's vocabulary.
        dict(name="rules_32_penalties", op="rules", batch=32, rows=248320, vocabulary=248077, history=4000, prompt=1500,
             bias=100, masked=False, penalties=True),
        # The largest batch, everything on.
        dict(name="rules_256_all", op="rules", batch=256, rows=151936, vocabulary=151936, history=2000, prompt=800,
             bias=300, masked=True, penalties=True),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "branch", "churn", "rules", "rules"])
    shape = rng.choice(["27b", "reference"])
    if op == "attention":
        c = dict(op=op, shape=shape, count=_log(rng, 1, 64), tokens=rng.choice([1, 1, rng.randint(2, 8), rng.randint(9, 32)]),
                 shared=rng.choice([0, _log(rng, 16, 32768), _log(rng, 16, 32768)]), own_min=rng.randint(0, 3),
                 own_max=_log(rng, 4, 4096), page=rng.choice([16, 32, 64, 128, 256]))
        most = work(listed()[4])
        while work(c)["flops"] > most["flops"] or work(c)["bytes"] > most["bytes"]:
            c["count"] = max(1, c["count"] * 3 // 4)
            c["tokens"] = max(1, c["tokens"] * 3 // 4)
            c["shared"] = c["shared"] * 7 // 8
        return c
    if op == "branch":
        page = rng.choice([16, 32, 64, 128])
        return dict(op=op, shape=shape, layers=rng.randint(1, LAYERS), page=page, parent=_log(rng, 1, 3900),
                    children=_log(rng, 1, 63), tokens=rng.choice([1, rng.randint(2, 5)]), others=_log(rng, 1, 100))
    if op == "churn":
        return dict(op=op, shape=shape, layers=rng.randint(1, LAYERS), page=rng.choice([16, 32, 64]),
                    length=_log(rng, 20, 2000), others=_log(rng, 1, 60))
    vocabulary = _log(rng, 1000, 140000)
    history = rng.choice([0, _log(rng, 1, 4000)])
    return dict(op=op, batch=_log(rng, 1, 256), rows=vocabulary + rng.choice([0, rng.randint(1, 300)]),
                vocabulary=vocabulary, history=history, prompt=rng.randint(0, history), bias=rng.choice([0, _log(rng, 1, 300)]),
                masked=rng.random() < 0.5, penalties=rng.random() < 0.8)


def _own_lengths(c):
    """Committed tokens past the prefix, by the case alone."""
    span = c["own_max"] - c["own_min"] + 1 if c["own_max"] >= c["own_min"] else 1
    return [c["own_min"] + (i * 7919 + 13) % span for i in range(c["count"])]


def work(c):
    if c["op"] == "attention":
        q_heads, kv_heads, d = HEADS[c["shape"]]
        lengths = [c["shared"] + o for o in _own_lengths(c)]
        positions = c["shared"] + sum(n - c["shared"] + c["tokens"] for n in lengths)
        rows = c["count"] * c["tokens"] * q_heads
        visible = sum(n + t + 1 for n in lengths for t in range(c["tokens"])) * q_heads
        return {"bytes": positions * kv_heads * d * 4 + rows * d * (2 + 4 + 2), "flops": 4 * visible * d}
    if c["op"] == "branch":
        _, kv_heads, d = HEADS[c["shape"]]
        row, tail, n = kv_heads * d, c["parent"] % c["page"], c["children"]
        pages = -(-c["parent"] // c["page"])
        return {"bytes": c["layers"] * row * (4 * tail * (1 + n) + 10 * n * c["tokens"]) + 4 * pages * (2 + n), "flops": 0}
    if c["op"] == "churn":
        _, kv_heads, d = HEADS[c["shape"]]
        row, pages = kv_heads * d, -(-c["length"] // c["page"])
        return {"bytes": 2 * c["layers"] * row * (8 * pages * c["page"] + 10 * c["length"]), "flops": 0}
    row = c["vocabulary"] * (8 + (1 / 8 if c["masked"] else 0)) + 4 * c["history"] + 8 * c["bias"]
    return {"bytes": int(c["batch"] * row), "flops": 4 * c["batch"] * c["vocabulary"]}


# ---- inputs -------------------------------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _normal(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(c, seed):
    state = {"attention": _prepare_attention, "branch": _prepare_branch, "churn": _prepare_churn,
             "rules": _prepare_rules}[c["op"]](c, _generator(seed))
    state["case"] = c
    if own:
        _handles(state)
    return state


def _prepare_attention(c, g):
    """Two layers of pages (the second is read), pages in no order, a prefix that may end inside a page."""
    q_heads, kv_heads, d = HEADS[c["shape"]]
    n, t, page, shared = c["count"], c["tokens"], c["page"], c["shared"]
    lengths = [shared + o for o in _own_lengths(c)]
    held = [-(-(length + t) // page) for length in lengths]
    common = shared // page
    pages = common + sum(h - common for h in held)
    order = torch.randperm(pages, generator=g, device=DEVICE).tolist()
    k = _normal((2, pages, page, kv_heads, d), g, torch.float16)
    v = _normal((2, pages, page, kv_heads, d), g, torch.float16)
    stride = max(held)
    table, references, at = [], [0] * pages, common
    for h in held:
        mine = order[:common] + order[at:at + h - common]
        at += h - common
        table.append(mine + [-1] * (stride - h))
        for p in mine:
            references[p] += 1
    rest = shared % page
    if rest:
        for row in table[1:]:
            for pool in (k, v):
                pool[:, row[common], :rest] = pool[:, table[0][common], :rest]
    return dict(k=k, v=v, table=_ints(table), lengths=_ints(lengths), references=_ints(references),
                query=_normal((n, t, q_heads, d), g, torch.float16), gate=_normal((n, t, q_heads, 2 * d), g),
                output=torch.zeros((n, t, q_heads, d), dtype=torch.float16, device=DEVICE))


def _prepare_branch(c, g):
    """Slot 0 the parent, slots 1..n its children to be, slot n + 1 another conversation; pages in no order."""
    _, kv_heads, d = HEADS[c["shape"]]
    n, page, layers = c["children"], c["page"], c["layers"]
    held = -(-c["parent"] // page)
    more = n * (1 + -(-(c["tokens"] + page) // page))
    pages = held + c["others"] + more
    order = torch.randperm(pages, generator=g, device=DEVICE).tolist()
    stride = max(held + -(-(c["tokens"] + page) // page), c["others"])
    none = [-1] * stride
    table = [(order[:held] + none)[:stride]] + [none] * n + [(order[held:held + c["others"]] + none)[:stride]]
    references = [0] * pages
    for p in order[:held + c["others"]]:
        references[p] = 1
    return dict(k=_normal((layers, pages, page, kv_heads, d), g, torch.float16),
                v=_normal((layers, pages, page, kv_heads, d), g, torch.float16), table=_ints(table),
                lengths=_ints([c["parent"]] + [0] * n + [c["others"] * page]), references=_ints(references),
                new_k=_normal((layers, n, c["tokens"], kv_heads, d), g, torch.float16),
                new_v=_normal((layers, n, c["tokens"], kv_heads, d), g),
                status=torch.zeros(1, dtype=torch.int32, device=DEVICE))


def _prepare_churn(c, g):
    """Slot 0 holds the first pages, slot 2 the last used ones, slot 1 (another conversation) those between."""
    _, kv_heads, d = HEADS[c["shape"]]
    page, layers, length = c["page"], c["layers"], c["length"]
    held = -(-length // page)
    live = 2 * held + c["others"]
    pages = live + 3
    middle = (held + torch.randperm(c["others"], generator=g, device=DEVICE)).tolist()
    stride = max(held, c["others"]) + 1
    none = [-1] * stride
    table = [(list(range(held)) + none)[:stride], (middle + none)[:stride],
             (list(range(held + c["others"], live)) + none)[:stride]]
    k, v = (_normal((layers, pages, page, kv_heads, d), g, torch.float16) for _ in range(2))
    if length % page:
        for pool in (k, v):
            pool[:, [held - 1, live - 1], length % page:] = 0
    return dict(k=k, v=v, table=_ints(table), lengths=_ints([length, c["others"] * page, length]),
                references=_ints([1] * live + [0] * 3), new_k=_normal((2, layers, 1, length, kv_heads, d), g, torch.float16),
                new_v=_normal((2, layers, 1, length, kv_heads, d), g),
                status=torch.zeros(1, dtype=torch.int32, device=DEVICE), live=torch.zeros(1, dtype=torch.int32, device=DEVICE))


def _prepare_rules(c, g):
    """Logits as a head gives them; histories in which few tokens come often; a third of the rows without a grammar."""
    batch, vocabulary = c["batch"], c["vocabulary"]
    uniform = lambda *shape: torch.rand(shape, generator=g, device=DEVICE)  # noqa: E731
    frequent = lambda *shape: (uniform(*shape).pow(4) * vocabulary).to(torch.int32).clamp_(0, vocabulary - 1)  # noqa: E731
    s = dict(logits=_normal((batch, c["rows"]), g) * 3, output=torch.zeros((batch, c["rows"]), device=DEVICE),
             tokens=torch.zeros(batch, dtype=torch.int32, device=DEVICE))
    if c["penalties"] and c["history"]:
        s["history"] = frequent(batch, c["history"])
        s["history_lengths"] = (c["history"] - (uniform(batch) * min(c["history"], 40)).to(torch.int32)).to(torch.int32)
        s["prompt_lengths"] = torch.full((batch,), c["prompt"], dtype=torch.int32, device=DEVICE)
        s["repetition"], s["presence"], s["frequency"] = 1 + uniform(batch) * 0.3, uniform(batch) * 0.5, uniform(batch) * 0.3
    if c["bias"]:
        s["bias_tokens"] = frequent(batch, c["bias"])
        s["bias_values"] = _normal((batch, c["bias"]), g) * 4
        s["bias_counts"] = (c["bias"] - (uniform(batch) * c["bias"] * 0.5).to(torch.int32)).to(torch.int32)
    if c["masked"]:
        words = -(-vocabulary // 32)
        masks = max(1, batch - batch // 3)
        s["allowed"] = (torch.randint(0, 1 << 32, (masks, words), generator=g, device=DEVICE)
                        & torch.randint(0, 1 << 32, (masks, words), generator=g, device=DEVICE)).to(torch.int32)
        rows = torch.arange(batch, device=DEVICE, dtype=torch.int32)
        s["allowed_rows"] = torch.where(rows < masks, rows, -1).to(torch.int32)
    return s


def _handles(s):
    """What a program keeps beside its tensors: the description of the cache or of the rules, and scratch."""
    import gfxinfer_amd as gx
    c = s["case"]
    scratch = lambda n: torch.empty(max(1, n), dtype=torch.uint8, device=DEVICE)  # noqa: E731
    if c["op"] == "rules":
        names = ("history", "history_lengths", "prompt_lengths", "repetition", "presence", "frequency", "bias_tokens",
                 "bias_values", "bias_counts", "allowed", "allowed_rows")
        s["rules"] = gx.LogitRules.of(**{k: s[k] for k in names if k in s})
        s["workspace"] = scratch(gx.logit_rules_workspace_bytes(c["vocabulary"], c["batch"]))
        return
    s["pages"] = gx.KvPages.of(s["k"], s["v"], s["table"], s["lengths"], s["references"])
    if c["op"] == "attention":
        s["workspace"] = scratch(gx.kv_pages_attention_workspace_bytes(s["pages"], c["count"], c["tokens"],
                                                                       HEADS[c["shape"]][0], c["shared"]))
    else:
        s["workspace"] = scratch(gx.kv_pages_workspace_bytes(s["pages"]))


# ---- one pass -----------------------------------------------------------------------------------------------


def run(state):
    return (_own_run if own else _plain_run)(state)


def _outputs(s):
    if s["case"]["op"] == "attention":
        return s["output"]
    if s["case"]["op"] == "rules":
        return {"logits": s["output"][:, :s["case"]["vocabulary"]], "tokens": s["tokens"]}
    return {"k": s["k"], "v": s["v"], "table": s["table"], "lengths": s["lengths"], "references": s["references"],
            "status": s["status"]}


def _own_run(s):
    import gfxinfer_amd as gx
    c = s["case"]
    if c["op"] == "attention":
        gx.launch_kv_pages_gated_attention(s["pages"], 1, s["query"], s["gate"], s["output"], range(c["count"]), c["tokens"],
                                           HEADS[c["shape"]][0], c["shared"], s["workspace"])
    elif c["op"] == "branch":
        children = range(1, c["children"] + 1)
        gx.launch_kv_pages_fork(s["pages"], 0, children)
        gx.launch_kv_pages_reserve(s["pages"], children, c["tokens"], s["status"], s["workspace"])
        for layer in range(c["layers"]):
            gx.launch_kv_pages_append(s["pages"], layer, s["new_k"][layer], s["new_v"][layer], children, c["tokens"])
        gx.launch_kv_pages_advance(s["pages"], children, c["tokens"])
    elif c["op"] == "churn":
        for turn, slot in enumerate((0, 2)):
            gx.launch_kv_pages_free(s["pages"], [slot])
            gx.launch_kv_pages_compact(s["pages"], s["live"], s["workspace"])
            gx.launch_kv_pages_reserve(s["pages"], [slot], c["length"], s["status"], s["workspace"])
            for layer in range(c["layers"]):
                gx.launch_kv_pages_append(s["pages"], layer, s["new_k"][turn, layer], s["new_v"][turn, layer], [slot],
                                          c["length"])
            gx.launch_kv_pages_advance(s["pages"], [slot], c["length"])
    else:
        gx.launch_logit_rules(s["logits"], s["rules"], s["output"], s["tokens"], s["workspace"], c["vocabulary"])
    return _outputs(s)


def _plain_run(s):
    c = s["case"]
    if c["op"] == "attention":
        _plain_attention(s, c)
    elif c["op"] == "branch":
        slots = torch.arange(1, c["children"] + 1, device=DEVICE)
        _plain_fork(s, c, 0, slots)
        _plain_reserve(s, c, slots, c["tokens"])
        _plain_append(s, c, slots, s["new_k"], s["new_v"])
        s["lengths"][slots] += c["tokens"]
    elif c["op"] == "churn":
        for turn, slot in enumerate((0, 2)):
            slots = torch.tensor([slot], device=DEVICE)
            _plain_free(s, slots)
            _plain_compact(s)
            _plain_reserve(s, c, slots, c["length"])
            _plain_append(s, c, slots, s["new_k"][turn], s["new_v"][turn])
            s["lengths"][slots] += c["length"]
    else:
        _plain_rules(s, c)
    return _outputs(s)


def _plain_attention(s, c):
    """Every sequence gathers its own pages: softmax(q k / sqrt(d)) v * sigmoid(gate), 32 bits throughout."""
    q_heads, kv_heads, d = HEADS[c["shape"]]
    n, t, page = c["count"], c["tokens"], c["page"]
    group, most = q_heads // kv_heads, c["shared"] + max(_own_lengths(c)) + t
    position = torch.arange(most, device=DEVICE)
    rows = s["table"][:, position // page].clamp(min=0).long() * page + position % page
    visible = s["lengths"][:, None] + torch.arange(1, t + 1, device=DEVICE)                      # [n, t]
    seen = (position < visible[:, -1:])[:, :, None, None]
    keys = s["k"][1].view(-1, kv_heads, d)[rows].float()
    values = torch.where(seen, s["v"][1].view(-1, kv_heads, d)[rows].float(), 0.0)
    query = s["query"].float().view(n, t, kv_heads, group, d).permute(0, 2, 1, 3, 4).reshape(n, kv_heads, t * group, d)
    scores = torch.matmul(query, keys.permute(0, 2, 3, 1).contiguous()) / math.sqrt(d)
    hidden = (position >= visible[:, :, None])[:, None, :, None, :]                              # [n, 1, t, 1, most]
    scores = scores.view(n, kv_heads, t, group, most).masked_fill_(hidden, -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(n, kv_heads, t * group, most), values.permute(0, 2, 1, 3).contiguous())
    out = (out.view(n, kv_heads, t, group, d) / total).permute(0, 2, 1, 3, 4).reshape(n, t, q_heads, d)
    s["output"].copy_(out * torch.sigmoid(s["gate"][..., d:]))


def _plain_free(s, slots):
    held = s["table"][slots]
    s["references"].scatter_add_(0, held.clamp(min=0).view(-1).long(), -(held >= 0).view(-1).int())
    s["table"][slots] = -1
    s["lengths"][slots] = 0


def _plain_fork(s, c, parent, slots):
    _plain_free(s, slots)
    column = torch.arange(s["table"].shape[1], device=DEVICE)
    shared = torch.where(column * c["page"] < s["lengths"][parent], s["table"][parent], -1)
    s["table"][slots] = shared
    s["references"].scatter_add_(0, shared.clamp(min=0).long(), (shared >= 0).int() * len(slots))
    s["lengths"][slots] = s["lengths"][parent].clone()


def _plain_reserve(s, c, slots, tokens):
    """Lowest free pages first; a shared partial tail page is copied, its last holder in the list keeps it."""
    page, n = c["page"], len(slots)
    table, length = s["table"][slots], s["lengths"][slots]
    column = torch.arange(table.shape[1], device=DEVICE)
    first, need = (length + page - 1) // page, (length + tokens + page - 1) // page
    start = first + ((table >= 0) & (column >= first[:, None]) & (column < need[:, None])).sum(1)
    partial = length % page > 0
    at = (length // page).long()[:, None]
    tail = torch.where(partial, table.gather(1, at)[:, 0], 0).long()
    same = (tail[:, None] == tail) & partial[:, None] & partial
    later = torch.triu(same, 1).any(1)
    holders = s["references"][tail]
    copied = partial & (holders > 1) & ((same.sum(1) < holders) | later)
    amount = (need - start).clamp(min=0) + copied
    offset = amount.cumsum(0) - amount
    free = torch.sort((s["references"] != 0).int(), stable=True)[1]
    target = torch.where(copied, free[offset.clamp(max=len(free) - 1)], tail)
    fresh = (column >= start[:, None]) & (column < need[:, None])
    rank = offset[:, None] + copied[:, None] + column - start[:, None]
    taken = free[rank.clamp(0, len(free) - 1)]
    table = torch.where(fresh, taken.int(), table)
    table.scatter_(1, at, torch.where(partial, target.int(), table.gather(1, at)[:, 0])[:, None])
    for pool in (s["k"], s["v"]):
        keep = (torch.arange(page, device=DEVICE) < (length % page)[:, None]) & copied[:, None]
        pool[:, target] = torch.where(keep[None, :, :, None, None], pool[:, tail], pool[:, target])
    s["references"].scatter_add_(0, tail, -copied.int())
    s["references"].scatter_add_(0, target, copied.int())
    s["references"].scatter_add_(0, taken.view(-1), fresh.view(-1).int())
    s["table"][slots] = table
    s["status"].zero_()


def _plain_append(s, c, slots, key, value):
    position = s["lengths"][slots][:, None] + torch.arange(key.shape[2], device=DEVICE)
    page = s["table"][slots].gather(1, (position // c["page"]).long()).long()
    s["k"][:, page, position % c["page"]] = key
    s["v"][:, page, position % c["page"]] = value.half()


def _plain_compact(s):
    """Used pages past the number of used pages move, in order, to the free pages before it, in order."""
    count = s["references"].shape[0]
    index = torch.arange(count, device=DEVICE)
    used = s["references"] != 0
    live = used.sum()
    movers = torch.sort((~(used & (index >= live))).int(), stable=True)[1]
    holes = torch.sort((used | (index >= live)).int(), stable=True)[1]
    moved = index < (used & (index >= live)).sum()
    source = torch.where(moved, movers, index)[moved]
    target = torch.where(moved, holes, index)[moved]
    for pool in (s["k"], s["v"]):
        pool[:, target] = pool[:, source]
    to = index.clone()
    to[source] = target
    s["references"][target] = s["references"][source]
    s["references"][source] = 0
    s["table"].copy_(torch.where(s["table"] >= 0, to[s["table"].clamp(min=0).long()].int(), s["table"]))
    s["live"].copy_(live)


def _plain_rules(s, c):
    batch, vocabulary = c["batch"], c["vocabulary"]
    x = s["logits"][:, :vocabulary].clone()
    if "history" in s:
        place = torch.arange(s["history"].shape[1], device=DEVICE)
        listed_ = (place < s["history_lengths"][:, None]).int()
        generated = listed_ * (place >= s["prompt_lengths"][:, None])
        history = s["history"].long()
        seen = torch.zeros((batch, vocabulary), dtype=torch.int32, device=DEVICE).scatter_add_(1, history, listed_)
        count = torch.zeros((batch, vocabulary), dtype=torch.int32, device=DEVICE).scatter_add_(1, history, generated.int())
        penalty = s["repetition"][:, None]
        x = torch.where(seen > 0, torch.where(x > 0, x / penalty, x * penalty), x)
        x = x - s["frequency"][:, None] * count
        x = torch.where(count > 0, x - s["presence"][:, None], x)
    if "bias_tokens" in s:
        place = torch.arange(1, s["bias_tokens"].shape[1] + 1, device=DEVICE).expand(batch, -1)
        place = torch.where(place <= s["bias_counts"][:, None], place, 0)
        last = torch.zeros((batch, vocabulary), dtype=torch.int64, device=DEVICE)
        last = last.scatter_reduce_(1, s["bias_tokens"].long(), place, "amax")
        x = torch.where(last > 0, x + s["bias_values"].gather(1, (last - 1).clamp(min=0)), x)
    index = torch.arange(vocabulary, device=DEVICE)
    if "allowed" in s:
        words = s["allowed"][s["allowed_rows"].clamp(min=0).long()]
        bit = (words[:, index // 32] >> (index % 32)) & 1
        x = torch.where((bit != 0) | (s["allowed_rows"] < 0)[:, None], x, -math.inf)
    s["output"][:, :vocabulary] = x
    top = x.amax(1, keepdim=True)
    s["tokens"].copy_(torch.where(x == top, index, vocabulary).amin(1))


# ---- the definitions in 64 bits -----------------------------------------------------------------------------


def exact(c, seed):
    s = prepare(c, seed)
    return {"attention": _exact_attention, "branch": _exact_branch, "churn": _exact_churn, "rules": _exact_rules}[c["op"]](s, c)


def _exact_attention(s, c):
    q_heads, kv_heads, d = HEADS[c["shape"]]
    out = torch.zeros((c["count"], c["tokens"], q_heads, d), dtype=torch.float64, device=DEVICE)
    for i, length in enumerate(s["lengths"].tolist()):
        pages = [p for p in s["table"][i].tolist() if p >= 0]
        key, value = (pool[1][pages].reshape(-1, kv_heads, d)[:length + c["tokens"]].double() for pool in (s["k"], s["v"]))
        for h in range(kv_heads):
            heads = slice(h * q_heads // kv_heads, (h + 1) * q_heads // kv_heads)
            for t in range(c["tokens"]):
                score = s["query"][i, t, heads].double() @ key[:length + t + 1, h].T.contiguous() * d ** -0.5
                out[i, t, heads] = torch.softmax(score, -1) @ value[:length + t + 1, h].contiguous()
    return out / (1 + torch.exp(-s["gate"][..., d:].double()))


def _exact_branch(s, c):
    """The same step, one child after another, with lists for the pages."""
    page, parent, tokens = c["page"], c["parent"], c["tokens"]
    k, v = s["k"].double(), s["v"].double()
    table, references, lengths = s["table"].tolist(), s["references"].tolist(), s["lengths"].tolist()
    held = table[0][:-(-parent // page)]
    free = [p for p, n in enumerate(references) if n == 0]
    for p in held:
        references[p] += c["children"]
    for child in range(1, c["children"] + 1):
        mine = list(held)
        if parent % page:
            mine[-1] = free.pop(0)
            k[:, mine[-1], :parent % page] = k[:, held[-1], :parent % page]
            v[:, mine[-1], :parent % page] = v[:, held[-1], :parent % page]
            references[held[-1]] -= 1
            references[mine[-1]] = 1
        while len(mine) * page < parent + tokens:
            mine.append(free.pop(0))
            references[mine[-1]] = 1
        for t in range(tokens):
            at = parent + t
            k[:, mine[at // page], at % page] = s["new_k"][:, child - 1, t].double()
            v[:, mine[at // page], at % page] = s["new_v"][:, child - 1, t].double()
        table[child] = (mine + [-1] * len(table[child]))[:len(table[child])]
        lengths[child] = parent + tokens
    return {"k": k, "v": v, "table": _ints(table), "lengths": _ints(lengths), "references": _ints(references), "status": None}


def _exact_churn(s, c):
    """Both sequences end where they began, with new rows; the pages behind the last used one keep what the moves left."""
    page, length = c["page"], c["length"]
    held = -(-length // page)
    last = held + c["others"]
    pools = []
    for pool, new in ((s["k"], s["new_k"]), (s["v"], s["new_v"])):
        pool = pool.double()
        for turn, start in enumerate((0, last)):
            rows = new[turn].double().reshape(c["layers"], length, *pool.shape[3:])
            for i in range(held):
                part = rows[:, i * page:(i + 1) * page]
                pool[:, start + i, :part.shape[1]] = part
        pools.append(pool)
    return {"k": pools[0], "v": pools[1], "table": s["table"], "lengths": s["lengths"], "references": s["references"],
            "status": None}


def _exact_rules(s, c):
    vocabulary = c["vocabulary"]
    out = s["logits"][:, :vocabulary].double()
    for b in range(c["batch"]):
        x = out[b]
        if "history" in s:
            tokens = s["history"][b, :int(s["history_lengths"][b])].long()
            seen = torch.bincount(tokens, minlength=vocabulary) > 0
            count = torch.bincount(tokens[c["prompt"]:], minlength=vocabulary).double()
            factor = s["repetition"][b].double()
            x = torch.where(seen & (x > 0), x / factor, torch.where(seen, x * factor, x))
            x = x - s["frequency"][b].double() * count - s["presence"][b].double() * (count > 0)
        if "bias_tokens" in s:
            added = dict(zip(*(s[k][b, :int(s["bias_counts"][b])].tolist() for k in ("bias_tokens", "bias_values"))))
            x = x.clone()
            x[list(added)] += torch.tensor(list(added.values()), dtype=torch.float64, device=DEVICE)
        if "allowed" in s and b < s["allowed"].shape[0]:
            bits = (s["allowed"][b][:, None] >> torch.arange(32, device=DEVICE)) & 1
            x = torch.where(bits.reshape(-1)[:vocabulary] > 0, x, torch.tensor(-math.inf, dtype=torch.float64, device=DEVICE))
        out[b] = x
    return {"logits": out, "tokens": None}
