"""Operators of long prompts in a bounded cache, as cases that can be timed and checked.

`attention`: gated GQA attention of ragged chunks of new tokens over K/V pages, with the log of each row's sum.
`weights`: the attention weight that each cached row receives from a chunk, added to what it has.
`evict`: room for new tokens, then back to a budget by dropping the rows of least weight.
`product`: a matrix product in 8-bit integers with a scale for each token and each output channel, quantizer included.

With `own` false the plain form runs, elementary torch operations in 32 bits; with `own` true the calls of
gfxinfer_amd.  `exact` states each operator once more, in 64 bits, sequence by sequence.
"""
import math

import torch

own = False

DEVICE = "cuda"
HEADS = {"27b": (40, 8, 128), "reference": (24, 4, 256)}   # query heads, KV heads, head size
LAYERS = 16                                                # full-attention layers of both shapes
TYPES = {"half": torch.float16, "brain": torch.bfloat16, "float": torch.float32}


def listed():
    return [
        # A decode step of eight conversations, some with a few drafted tokens: latency counts.
        dict(name="attention_8_decode", op="attention", shape="27b", page=16, count=8, chunks=0, chunk=1, small=4,
             length_min=0, length_max=600),
        # An ordinary serving step: one prompt's chunk beside 31 sequences that decode.
        dict(name="attention_32_mixed", op="attention", shape="27b", page=64, count=32, chunks=1, chunk=509, small=1,
             length_min=200, length_max=4090),
        # Prompts of four users, late in their conversations, 256-wide heads.
        dict(name="attention_4_prompts", op="attention", shape="reference", page=32, count=4, chunks=4, chunk=300, small=1,
             length_min=1500, length_max=6000),
        # A chunk near the end of a long document.
        dict(name="attention_1_document", op="attention", shape="27b", page=128, count=1, chunks=1, chunk=2048, small=1,
             length_min=30000, length_max=30000),
        # Weights while 16 sequences decode.
        dict(name="weights_16_decode", op="weights", shape="reference", page=16, count=16, chunks=0, chunk=1, small=1,
             length_min=2, length_max=4090),
        # Weights of a document's chunk.
        dict(name="weights_1_document", op="weights", shape="27b", page=64, count=1, chunks=1, chunk=2048, small=1,
             length_min=8000, length_max=8000),
        # Four decoding sequences at a small budget: every step drops one row each.
        dict(name="evict_4_decode", op="evict", shape="27b", layers=LAYERS, page=16, count=4, tokens=1, budget=500, first=4,
             recent=64, shared=0),
        # Eight prompts fed in chunks; their first pages are shared at first.
        dict(name="evict_8_chunks", op="evict", shape="reference", layers=LAYERS, page=64, count=8, tokens=512, budget=2048,
             first=16, recent=400, shared=300),
        # The output projection for one token.
        dict(name="product_1_token", op="product", tokens=1, rows=5120, columns=5120, input="half", output="float"),
        # An up projection for a decode batch of odd size.
        dict(name="product_37_tokens", op="product", tokens=37, rows=17408, columns=5120, input="half", output="float"),
        # A down projection for a prompt's chunk.
        dict(name="product_509_tokens", op="product", tokens=509, rows=5120, columns=17408, input="half", output="float"),
        # An up projection for many prompts at once.
        dict(name="product_4096_tokens", op="product", tokens=4096, rows=17408, columns=5120, input="half", output="half"),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "weights", "evict", "product", "product", "product"])
    shape = rng.choice(["27b", "reference"])
    if op in ("attention", "weights"):
        count = _log(rng, 1, 48)
        c = dict(op=op, shape=shape, page=rng.choice([16, 32, 64, 128, 256]), count=count,
                 chunks=rng.choice([0, 1, rng.randint(1, count)]), chunk=_log(rng, 9, 2048), small=rng.choice([1, rng.randint(2, 8)]),
                 length_min=rng.choice([0, rng.randint(1, 40)]), length_max=_log(rng, 41, 30000))
        most = listed()[3 if op == "attention" else 5]
        room = lambda x: x["count"] * max(_tokens(x)) * (max(_lengths(x)) + max(_tokens(x)))  # noqa: E731  (the padded scores)
        while room(c) > room(most) or work(c)["bytes"] > 2 ** 30:
            c["length_max"] = max(41, c["length_max"] * 3 // 4)
            c["chunk"] = max(1, c["chunk"] * 3 // 4)
            c["count"] = max(1, c["count"] * 3 // 4)
            c["chunks"] = min(c["chunks"], c["count"])
        return c
    if op == "evict":
        budget = _log(rng, 32, 2500)
        return dict(op=op, shape=shape, layers=rng.randint(1, LAYERS), page=rng.choice([16, 32, 64, 128]), count=_log(rng, 1, 8),
                    tokens=_log(rng, 1, 600), budget=budget, first=rng.randint(0, min(16, budget // 4)),
                    recent=rng.randint(0, budget // 2), shared=rng.choice([0, 0, rng.randint(0, budget // 2)]))
    return dict(op=op, tokens=_log(rng, 1, 4096), rows=_log(rng, 256, 17408), columns=16 * _log(rng, 16, 320),
                input=rng.choice(["half", "half", "brain", "float"]), output=rng.choice(["half", "float"]))


def _spread(low, high, i):
    return low + (i * 7919 + 13) % (high - low + 1)


def _lengths(c):
    """Committed tokens of each sequence, by the case alone."""
    return [_spread(c["length_min"], c["length_max"], i) for i in range(c["count"])]


def _tokens(c):
    """New tokens of each sequence: chunks first, then a few each."""
    return [c["chunk"] - i * 37 % (c["chunk"] // 8 + 1) if i < c["chunks"] else _spread(1, c["small"], i) for i in range(c["count"])]


def work(c):
    if c["op"] in ("attention", "weights"):
        q_heads, kv_heads, d = HEADS[c["shape"]]
        both = list(zip(_lengths(c), _tokens(c)))
        positions = sum(n + t for n, t in both)
        rows = sum(t for _, t in both) * q_heads
        visible = sum(n * t + t * (t + 1) // 2 for n, t in both) * q_heads
        if c["op"] == "attention":
            return {"bytes": positions * kv_heads * d * 4 + rows * (d * (2 + 4 + 2) + 4), "flops": 4 * visible * d}
        return {"bytes": positions * (kv_heads * d * 2 + 8) + rows * (d * 2 + 4), "flops": 2 * visible * d}
    if c["op"] == "evict":
        _, kv_heads, d = HEADS[c["shape"]]
        moved = c["count"] * min(c["tokens"], c["recent"])
        return {"bytes": moved * c["layers"] * kv_heads * d * 8 + c["count"] * (c["budget"] + c["tokens"]) * 8, "flops": 0}
    size = {"half": 2, "brain": 2, "float": 4}
    return {"bytes": c["columns"] * (c["rows"] + c["tokens"] * size[c["input"]]) + 4 * (c["rows"] + c["tokens"])
            + c["rows"] * c["tokens"] * size[c["output"]], "flops": 2 * c["tokens"] * c["rows"] * c["columns"]}


# ---- inputs -------------------------------------------------------------------------------------------------


def _normal(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(c, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    state = {"attention": _prepare_attention, "weights": _prepare_weights, "evict": _prepare_evict,
             "product": _prepare_product}[c["op"]](c, g)
    state["case"] = c
    if own:
        _handles(state)
    return state


def _prepare_attention(c, g):
    """Two layers of pages in no order (the second is read); the chunks' own rows are appended already."""
    q_heads, kv_heads, d = HEADS[c["shape"]]
    lengths, tokens, page = _lengths(c), _tokens(c), c["page"]
    held = [-(-(n + t) // page) for n, t in zip(lengths, tokens)]
    pages = sum(held)
    order = torch.randperm(pages, generator=g, device=DEVICE).tolist()
    table, references, at = [], [1] * pages, 0
    for h in held:
        table.append(order[at:at + h] + [-1] * (max(held) - h))
        at += h
    rows = sum(tokens)
    return dict(k=_normal((2, pages, page, kv_heads, d), g, torch.float16), v=_normal((2, pages, page, kv_heads, d), g, torch.float16),
                table=_ints(table), lengths=_ints(lengths), references=_ints(references), tokens=_ints(tokens),
                query=_normal((rows, q_heads, d), g, torch.float16), gate=_normal((rows, q_heads, 2 * d), g),
                output=torch.zeros((rows, q_heads, d), dtype=torch.float16, device=DEVICE),
                sums=torch.zeros((rows, q_heads), device=DEVICE))


def _prepare_weights(c, g):
    """The same after the attention: its sums are there, and rows that have received weight before."""
    s = _prepare_attention(c, g)
    shape = (c["count"], s["table"].shape[1] * c["page"])
    s["case"] = c
    s["sums"] = _padded(s, c, lambda x: torch.logsumexp(x, -1))
    s["weight"] = _normal(shape, g).square_()
    place = torch.arange(shape[1], device=DEVICE)
    s["weight"] *= place < s["lengths"][:, None]
    s["position"], s["dropped"] = place.int().repeat(c["count"], 1), torch.zeros(c["count"], dtype=torch.int32, device=DEVICE)
    return s


def _prepare_evict(c, g):
    """Sequences at their budget; the first pages of all are the same ones where something is shared."""
    _, kv_heads, d = HEADS[c["shape"]]
    n, page, budget = c["count"], c["page"], c["budget"]
    common, held = c["shared"] // page if n > 1 else 0, -(-budget // page)
    stride = -(-(budget + c["tokens"]) // page)
    pages = common + n * (stride + common)
    order = torch.randperm(pages, generator=g, device=DEVICE).tolist()
    table, references = [], [0] * pages
    for i in range(n):
        at = common + i * (held - common)
        mine = order[:common] + order[at:at + held - common]
        table.append(mine + [-1] * (stride - held))
        for p in mine:
            references[p] += 1
    return dict(k=_normal((c["layers"], pages, page, kv_heads, d), g, torch.float16),
                v=_normal((c["layers"], pages, page, kv_heads, d), g, torch.float16), table=_ints(table),
                lengths=_ints([budget] * n), references=_ints(references),
                weight=_normal((n, stride * page), g).exp_(),
                position=torch.arange(stride * page, device=DEVICE, dtype=torch.int32).repeat(n, 1),
                dropped=torch.zeros(n, dtype=torch.int32, device=DEVICE),
                status=torch.zeros(1, dtype=torch.int32, device=DEVICE))


def _prepare_product(c, g):
    """Activations with a few large channels, as hidden states have; weights in 8 bits, quantized beforehand."""
    x = _normal((c["tokens"], c["columns"]), g)
    x *= _normal((c["columns"],), g).mul_(0.5).exp_()
    w = _normal((c["rows"], c["columns"]), g)
    scale = w.abs().amax(1) / 127
    return dict(x=x.to(TYPES[c["input"]]), w=(w / scale[:, None]).round_().to(torch.int8), w_scale=scale * 0.02,
                output=torch.zeros((c["tokens"], c["rows"]), dtype=TYPES[c["output"]], device=DEVICE))


def _handles(s):
    """What a program keeps beside its tensors: descriptions of the cache and its weights, host lists, scratch."""
    import gfxinfer_amd as gx
    c = s["case"]
    scratch = lambda n: torch.empty(max(1, n), dtype=torch.uint8, device=DEVICE)  # noqa: E731
    if c["op"] == "product":
        s["codes"] = torch.empty((c["tokens"], c["columns"]), dtype=torch.int8, device=DEVICE)
        s["x_scale"] = torch.empty(c["tokens"], device=DEVICE)
        s["workspace"] = scratch(gx.w8a8_gemm_workspace_bytes(c["rows"], c["columns"], c["tokens"]))
        return
    s["pages"] = gx.KvPages.of(s["k"], s["v"], s["table"], s["lengths"], s["references"])
    s["listed"] = list(range(c["count"]))
    if c["op"] != "attention":
        s["weights"] = gx.KvWeights.of(s["pages"], s["weight"], s["position"], s["dropped"])
    if c["op"] == "evict":
        s["workspace"] = scratch(max(gx.kv_pages_workspace_bytes(s["pages"]),
                                     gx.kv_pages_evict_workspace_bytes(s["pages"], c["count"], c["budget"])))
        return
    s["host_tokens"] = _tokens(c)
    size = gx.kv_pages_chunk_attention_workspace_bytes if c["op"] == "attention" else gx.kv_weights_workspace_bytes
    s["workspace"] = scratch(size(s["pages"], s["host_tokens"], HEADS[c["shape"]][0]))


# ---- one pass -----------------------------------------------------------------------------------------------


def run(state):
    return (_own_run if own else _plain_run)(state)


def _outputs(s):
    op = s["case"]["op"]
    if op == "attention":
        return {"output": s["output"], "sums": s["sums"]}
    if op == "weights":
        return s["weight"]
    if op == "evict":
        kept = slice(0, s["case"]["budget"])
        return {"k": s["k"], "v": s["v"], "table": s["table"], "lengths": s["lengths"], "references": s["references"],
                "weight": s["weight"][:, kept], "position": s["position"][:, kept], "dropped": s["dropped"], "status": s["status"]}
    return s["output"]


def _own_run(s):
    import gfxinfer_amd as gx
    c = s["case"]
    if c["op"] == "attention":
        gx.launch_kv_pages_chunk_attention(s["pages"], 1, s["query"], s["gate"], s["output"], s["sums"], s["listed"],
                                           s["host_tokens"], HEADS[c["shape"]][0], s["workspace"])
    elif c["op"] == "weights":
        gx.launch_kv_weights_add(s["pages"], s["weights"], 1, s["query"], s["sums"], s["listed"], s["host_tokens"],
                                 HEADS[c["shape"]][0], s["workspace"])
    elif c["op"] == "evict":
        tokens = [c["tokens"]] * c["count"]
        gx.launch_kv_pages_reserve(s["pages"], s["listed"], c["tokens"], s["status"], s["workspace"])
        gx.launch_kv_weights_begin(s["pages"], s["weights"], s["listed"], tokens)
        gx.launch_kv_pages_advance(s["pages"], s["listed"], c["tokens"])
        gx.launch_kv_pages_evict(s["pages"], s["weights"], s["listed"], c["budget"], c["first"], c["recent"], s["status"],
                                 s["workspace"])
    else:
        gx.launch_quantize_rows_i8(s["x"], s["codes"], s["x_scale"])
        gx.launch_w8a8_gemm(s["w"], s["w_scale"], s["codes"], s["x_scale"], s["output"], s["workspace"])
    return _outputs(s)


def _plain_run(s):
    c = s["case"]
    if c["op"] == "attention":
        _plain_attention(s, c)
    elif c["op"] == "weights":
        _plain_weights(s, c)
    elif c["op"] == "evict":
        _plain_room(s, c)
        _plain_evict(s, c)
    else:
        x = s["x"].float()
        scale = x.abs().amax(1, keepdim=True) / 127
        codes = (x.double() / scale.double()).round().float().clamp(-127, 127)   # 64 bits: quotients next to a half
        s["output"].copy_(torch.matmul(codes, s["w"].float().T) * scale * s["w_scale"])
    return _outputs(s)


def _places(s):
    """Sequence and token of every packed row."""
    tokens = s["tokens"].long()
    sequence = torch.repeat_interleave(torch.arange(len(tokens), device=DEVICE), tokens, output_size=s["query"].shape[0])
    return sequence, torch.arange(s["query"].shape[0], device=DEVICE) - (tokens.cumsum(0) - tokens)[sequence]


def _scores(s, c):
    """Scaled scores [sequence, KV head, token, head in group, position], padded to the longest, -inf where unseen."""
    q_heads, kv_heads, d = HEADS[c["shape"]]
    n, page, group = c["count"], c["page"], q_heads // kv_heads
    sequence, token = _places(s)
    t, most = max(_tokens(c)), max(a + b for a, b in zip(_lengths(c), _tokens(c)))
    position = torch.arange(most, device=DEVICE)
    rows = s["table"][:, position // page].clamp(min=0).long() * page + position % page
    query = torch.zeros((n, t, q_heads, d), device=DEVICE)
    query[sequence, token] = s["query"].float()
    query = query.view(n, t, kv_heads, group, d).permute(0, 2, 1, 3, 4).reshape(n, kv_heads, t * group, d)
    keys = s["k"][1].view(-1, kv_heads, d)[rows].float().permute(0, 2, 3, 1).contiguous()
    scores = torch.matmul(query, keys).div_(math.sqrt(d)).view(n, kv_heads, t, group, most)
    hidden = position > s["lengths"][:, None, None] + torch.arange(t, device=DEVICE)[:, None]
    return scores.masked_fill_(hidden[:, None, :, None], -math.inf), rows, sequence, token


def _padded(s, c, f):
    """f of each row's scores, packed: [row, query head]."""
    scores, _, sequence, token = _scores(s, c)
    x = f(scores).permute(0, 2, 1, 3)[sequence, token]
    return x.reshape(x.shape[0], -1).contiguous()


def _plain_attention(s, c):
    """Every sequence gathers its own pages: softmax(q k / sqrt(d)) v * sigmoid(gate), 32 bits throughout."""
    q_heads, kv_heads, d = HEADS[c["shape"]]
    scores, rows, sequence, token = _scores(s, c)
    n, _, t, group, most = scores.shape
    top = scores.amax(-1, keepdim=True)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    seen = (torch.arange(most, device=DEVICE) < (s["lengths"] + s["tokens"])[:, None])[:, :, None, None]
    values = torch.where(seen, s["v"][1].view(-1, kv_heads, d)[rows].float(), 0.0).permute(0, 2, 1, 3).contiguous()
    out = torch.matmul(weights.view(n, kv_heads, t * group, most), values).view(n, kv_heads, t, group, d) / total
    out = out.permute(0, 2, 1, 3, 4)[sequence, token].reshape(-1, q_heads, d)
    s["output"].copy_(out * torch.sigmoid(s["gate"][..., d:]))
    s["sums"].copy_((top + total.log())[..., 0].permute(0, 2, 1, 3)[sequence, token].reshape(-1, q_heads))


def _plain_weights(s, c):
    q_heads, kv_heads, _ = HEADS[c["shape"]]
    scores, _, sequence, token = _scores(s, c)
    n, _, t, group, most = scores.shape
    sums = torch.full((n, t, q_heads), math.inf, device=DEVICE)
    sums[sequence, token] = s["sums"]
    sums = sums.view(n, t, kv_heads, group).permute(0, 2, 1, 3)[..., None]
    s["weight"][:, :most] += scores.sub_(sums).exp_().sum((1, 2, 3))


def _plain_room(s, c):
    """Pages for `tokens` more rows of each sequence, lowest free pages first; the rows begin without weight."""
    page, tokens = c["page"], c["tokens"]
    column = torch.arange(s["table"].shape[1], device=DEVICE)
    length = s["lengths"][:, None]
    fresh = (s["table"] < 0) & (column < (length + tokens + page - 1) // page)
    free = torch.sort((s["references"] != 0).int(), stable=True)[1]
    taken = free[(fresh.view(-1).cumsum(0) - 1).clamp(min=0)].view(fresh.shape)
    s["references"].scatter_add_(0, taken.view(-1), fresh.view(-1).int())
    s["table"].copy_(torch.where(fresh, taken.int(), s["table"]))
    row = torch.arange(s["weight"].shape[1], device=DEVICE)
    new = (row >= length) & (row < length + tokens)
    s["weight"].masked_fill_(new, 0)
    s["position"].copy_(torch.where(new, (row + s["dropped"][:, None]).int(), s["position"]))
    s["lengths"] += tokens


def _plain_evict(s, c):
    """The heaviest rows stay, the first and the last positions in any case; kept rows past the budget fill the holes before it."""
    page, budget, most = c["page"], c["budget"], s["weight"].shape[1]
    n, length = c["count"], s["lengths"][:, None]
    over = length > budget
    row = torch.arange(most, device=DEVICE)
    there = row < length
    fixed = (s["position"] < c["first"]) | (s["position"] >= length + s["dropped"][:, None] - c["recent"])
    value = torch.where(there, torch.where(fixed, math.inf, s["weight"]), -math.inf)
    rank = torch.sort(torch.sort(value, dim=1, descending=True, stable=True)[1], dim=1)[1]
    kept = there & ((rank < budget) | ~over)
    hole = ~kept & (row < budget) & over
    mover = kept & (row >= budget) & over
    # Holes in pages that others hold too: private copies, sequence by sequence, page by page.
    column = torch.arange(s["table"].shape[1], device=DEVICE)
    held = s["table"].clamp(min=0).long()
    copied = hole.view(n, -1, page).any(-1) & (s["table"] >= 0) & (s["references"][held] > 1)
    free = torch.sort((s["references"] != 0).int(), stable=True)[1]
    to = free[(copied.view(-1).cumsum(0) - 1).clamp(min=0)].view(copied.shape)
    table = torch.where(copied, to, held)
    at = lambda t, i, r: t[i, r // page] * page + r % page  # noqa: E731
    i, r = torch.nonzero(copied[:, row // page] & kept & (row < budget), as_tuple=True)
    source, target = at(held, i, r), at(table, i, r)
    # The k-th mover of a sequence goes to its k-th hole.
    (i, a), (_, b) = torch.nonzero(mover, as_tuple=True), torch.nonzero(hole, as_tuple=True)
    source, target = torch.cat([source, at(held, i, a)]), torch.cat([target, at(table, i, b)])
    for pool in (s["k"], s["v"]):
        flat = pool.view(pool.shape[0], -1, *pool.shape[3:])
        flat[:, target] = flat[:, source]
    for x in (s["weight"], s["position"]):
        x[i, b] = x[i, a]
    s["references"].scatter_add_(0, held.view(-1), -copied.view(-1).int())
    s["references"].scatter_add_(0, to.view(-1), copied.view(-1).int())
    past = (column >= -(-budget // page)) & (s["table"] >= 0) & over
    s["references"].scatter_add_(0, held.view(-1), -past.view(-1).int())
    s["table"].copy_(torch.where(past, -1, torch.where(copied, to.int(), s["table"])))
    s["dropped"] += (s["lengths"] - budget).clamp(min=0)
    s["lengths"].clamp_(max=budget)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------


def exact(c, seed):
    s = prepare(c, seed)
    return {"attention": _exact_attention, "weights": _exact_weights, "evict": _exact_evict, "product": _exact_product}[c["op"]](s, c)


def _exact_rows(s, c):
    """Per sequence and KV head: index of the sequence, rows of q, scaled scores of one head after another, values."""
    q_heads, kv_heads, d = HEADS[c["shape"]]
    group, at = q_heads // kv_heads, 0
    for i, (n, t) in enumerate(zip(_lengths(c), _tokens(c))):
        pages = [p for p in s["table"][i].tolist() if p >= 0]
        seen = torch.arange(n + t, device=DEVICE) <= n + torch.arange(t, device=DEVICE)[:, None]
        for h in range(kv_heads):
            key, value = (pool[1, pages, :, h].reshape(-1, d)[:n + t].double() for pool in (s["k"], s["v"]))
            for head in range(h * group, (h + 1) * group):
                score = s["query"][at:at + t, head].double() @ key.T.contiguous() * d ** -0.5
                yield i, slice(at, at + t), head, torch.where(seen, score, -math.inf), value
        at += t


def _exact_attention(s, c):
    out, sums = torch.zeros_like(s["output"], dtype=torch.float64), torch.zeros_like(s["sums"], dtype=torch.float64)
    d = out.shape[2]
    for _, rows, head, score, value in _exact_rows(s, c):
        out[rows, head] = torch.softmax(score, -1) @ value / (1 + torch.exp(-s["gate"][rows, head, d:].double()))
        sums[rows, head] = torch.logsumexp(score, -1)
    return {"output": out, "sums": sums}


def _exact_weights(s, c):
    weight = s["weight"].double()
    for i, rows, head, score, _ in _exact_rows(s, c):
        weight[i, :score.shape[1]] += torch.exp(score - s["sums"][rows, head].double()[:, None]).sum(0)
    return weight


def _exact_evict(s, c):
    """One sequence after another, with lists."""
    page, budget, tokens = c["page"], c["budget"], c["tokens"]
    k, v, weight = s["k"].double(), s["v"].double(), s["weight"].double()
    table, references = s["table"].tolist(), s["references"].tolist()
    position, dropped = s["position"].tolist(), s["dropped"].tolist()
    free = [p for p, n in enumerate(references) if n == 0]
    for i in range(c["count"]):
        for column in range(-(-(budget + tokens) // page)):
            if table[i][column] < 0:
                table[i][column] = free.pop(0)
                references[table[i][column]] = 1
        weight[i, budget:budget + tokens] = 0
        position[i][budget:budget + tokens] = [j + dropped[i] for j in range(budget, budget + tokens)]
    before, moves = list(references), []
    for i in range(c["count"]):
        end = budget + tokens + dropped[i]
        w = weight[i].tolist()
        order = sorted(range(budget + tokens), key=lambda j: (not (position[i][j] < c["first"] or position[i][j] >= end - c["recent"]), -w[j], j))
        kept = sorted(order[:budget])
        below = set(kept)
        holes, movers = [j for j in range(budget) if j not in below], [j for j in kept if j >= budget]
        old = list(table[i])
        for column in sorted({j // page for j in holes}):
            if before[old[column]] > 1:
                references[old[column]] -= 1
                table[i][column] = free.pop(0)
                references[table[i][column]] = 1
                moves += [(old[column], j % page, table[i][column], j % page) for j in kept if j // page == column and j < budget]
        for j, m in zip(holes, movers):
            moves.append((old[m // page], m % page, table[i][j // page], j % page))
            weight[i, j] = w[m]
            position[i][j] = position[i][m]
        for column in range(-(-budget // page), len(old)):
            if old[column] >= 0:
                references[old[column]] -= 1
                table[i][column] = -1
        dropped[i] += tokens
    if moves:
        a, b, e, f = (torch.tensor(x, device=DEVICE) for x in zip(*moves))
        for pool in (k, v):
            pool[:, e, f] = pool[:, a, b]
    return {"k": k, "v": v, "table": _ints(table), "lengths": s["lengths"], "references": _ints(references),
            "weight": weight[:, :budget], "position": _ints(position)[:, :budget], "dropped": _ints(dropped), "status": None}


def _exact_product(s, c):
    x = s["x"].double()
    scale = (s["x"].float().abs().amax(1, keepdim=True) / 127).double()
    codes = (x / scale).round().clamp(-127, 127)
    return codes @ s["w"].double().T.contiguous() * scale * s["w_scale"].double()
