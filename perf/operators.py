"""Performance cases of the streaming-generation operators: attention with a
sliding window and sinks over a paged cache (one new token a request, and a
chunk of a prompt), page moves with the block tables that follow them, and log
probabilities with entropy and top alternatives.

A case is one call as a server makes it.  `own` chooses between the plain form
(elementary torch operations in 32 bits) and the package's entry points.
Geometry is that of the benchmark (32 heads of 128, 8 or 32 K/V heads, pages
of 16, vocabulary 32000), of the tests (head dim 64, odd pages and widths) and
generic.

kinds:
  decode  windowed attention of one new token for each request of a batch
  chunk   windowed attention of a chunk of one prompt over its paged cache
  moves   pages copied inside the pools of several layers, and the tables
          rebuilt: "fork" (children take their parents' rows and a copy of the
          partly filled last page) and "compact" (live pages move to the front)
  score   log probability of a given token per row of logits, the row's
          entropy and its most probable tokens
"""
from __future__ import annotations

import importlib
import math
import random

import torch

own = False
F16 = torch.float16


def _tmc():
    return importlib.import_module("aicompiler-test_amd")


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one chat user's token with a short context: every position is still
        # inside the window, and latency is what counts
        dict(name="decode_b1_short", kind="decode", batch=1, active=1, heads=32, kv_heads=32,
             dim=128, page=16, low=300, high=300, window=1024, sinks=4, trimmed=False),
        # the benchmark's batch-16 grouped-query decode, some requests past the window
        dict(name="decode_b16_gqa", kind="decode", batch=16, active=16, heads=32, kv_heads=8,
             dim=128, page=16, low=65, high=4096, window=1024, sinks=4, trimmed=False),
        # a small model's server: head dim 64, odd page size, a padded batch
        dict(name="decode_b24_d64", kind="decode", batch=24, active=21, heads=32, kv_heads=8,
             dim=64, page=12, low=40, high=2000, window=500, sinks=7, trimmed=False),
        # one very long stream whose passed pages were given back
        dict(name="decode_b1_stream", kind="decode", batch=1, active=1, heads=32, kv_heads=8,
             dim=128, page=16, low=100000, high=100000, window=8192, sinks=64, trimmed=True),
        # a busy server of long streams
        dict(name="decode_b64_stream", kind="decode", batch=64, active=64, heads=32, kv_heads=8,
             dim=128, page=16, low=500, high=16384, window=2048, sinks=4, trimmed=True),
        # a middle chunk of a long prompt, grouped-query, short window
        dict(name="chunk_512_gqa", kind="chunk", rows=512, active=512, start=3584, heads=32,
             kv_heads=8, dim=128, page=16, window=1024, sinks=4, trimmed=True),
        # the odd end of a prompt on a head dim 64 model, padded to its bucket
        dict(name="chunk_203_d64", kind="chunk", rows=256, active=203, start=700, heads=32,
             kv_heads=8, dim=64, page=12, window=100, sinks=7, trimmed=False),
        # a full-size chunk of a long prompt, one K/V head per query head
        dict(name="chunk_2048_mha", kind="chunk", rows=2048, active=2048, start=2048, heads=32,
             kv_heads=32, dim=128, page=16, window=2048, sinks=16, trimmed=False),
        # best-of-n sampling: eight requests fork into four continuations each
        dict(name="fork_8x4", kind="moves", style="fork", layers=32, parents=8, children=4,
             heads=8, dim=128, page=16, pages=320, low=60, high=500),
        # a fragmented cache is packed to the front of its pools
        dict(name="compact_4k", kind="moves", style="compact", layers=4, rows=32, live=0.5,
             heads=8, dim=128, page=16, pages=4096),
        # the chosen tokens of a decode step, with alternatives
        dict(name="score_b16", kind="score", rows=16, vocab=32000, top=20, type="f32", masked=0.1,
             padded=False),
        # a prompt scored: every row's next token, odd vocabulary
        dict(name="score_2048", kind="score", rows=2048, vocab=32003, top=5, type="f32", masked=0.0,
             padded=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random):
    """One more case of the ranges above: batches of 1 to 64 tokens, windows
    of 1 to 8192 positions in caches of up to 131072, chunks of 1 to 2048
    rows, 1 to 32 layers of pools, vocabularies of 100 to 160000."""
    kind = rng.choice(["decode", "decode", "chunk", "chunk", "moves", "score"])
    group = rng.choice([1, 2, 4, 4, 8])
    geometry = dict(heads=32, kv_heads=32 // group, dim=rng.choice([64, 128, 128]),
                    page=rng.choice([16, 16, 32, 64, 12, 1]))
    sinks = rng.choice([0, 1, 4, 4, _log(rng, 5, 200)])
    if kind == "decode":
        batch = _log(rng, 1, 64)
        most = 64 * 2048 * 8 // (batch * geometry["kv_heads"]) - sinks - 1
        window = _log(rng, 1, min(8192, most))
        high = _log(rng, max(16, window // 2), 16 * min(window + 100, 8192))
        trimmed = rng.random() < 0.5 or batch * high > 200000
        return dict(kind=kind, batch=batch, active=max(1, batch - rng.choice([0, 0, 3])),
                    low=max(1, high // rng.randint(1, 20)), high=high, window=window, sinks=sinks,
                    trimmed=trimmed, **geometry)
    if kind == "chunk":
        rows = _log(rng, 1, 2048)
        window = _log(rng, 1, 2048)
        return dict(kind=kind, rows=rows, active=max(1, rows - rng.choice([0, 0, rows // 5])),
                    start=rng.choice([0, rng.randint(1, 2048), rng.randint(1, 30000)]),
                    window=window, sinks=sinks, trimmed=rng.random() < 0.5, **geometry)
    if kind == "moves":
        layers = _log(rng, 1, 32)
        heads, dim, page = rng.choice([1, 4, 8, 32]), geometry["dim"], rng.choice([16, 32, 12, 1])
        page_bytes = 2 * heads * dim * page
        if rng.random() < 0.5:
            parents, children = _log(rng, 1, 16), rng.randint(1, 8)
            high = page * rng.randint(1, 30)
            pages = parents * (children + high // page) + 8
            return dict(kind=kind, style="fork", layers=layers, parents=parents,
                        children=children, heads=heads, dim=dim, page=page, pages=pages,
                        low=max(1, high // 4), high=high)
        most = 4 * 4096 * 2 * 8 * 128 * 16 // (layers * page_bytes)
        return dict(kind=kind, style="compact", layers=layers, rows=_log(rng, 1, 64),
                    live=rng.choice([0.2, 0.5, 0.8]), heads=heads, dim=dim, page=page,
                    pages=_log(rng, 64, max(65, min(8192, most))))
    vocab = _log(rng, 100, 160000)
    rows = _log(rng, 1, min(4096, 2048 * 32003 // vocab))
    return dict(kind=kind, rows=rows, vocab=vocab, top=rng.choice([0, 1, 5, 10, 20]),
                type=rng.choice(["f32", "f32", "f16"]), masked=rng.choice([0.0, 0.0, 0.3]),
                padded=rng.random() < 0.5)


# ---------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=F16)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _spread(low, high, count):
    """`count` lengths evenly over [low, high], the longest at high."""
    if count == 1:
        return [high]
    return [low + (high - low) * i // (count - 1) for i in range(count)]


def _lengths(case, seed):
    lengths = _spread(case["low"], case["high"], case["batch"])
    random.Random(seed * 7919 + 13).shuffle(lengths)
    return lengths


def _held(case, first, end):
    """Logical pages of a cache of `end` positions whose earliest query sits at
    position first: those that the window or the sinks still reach where the
    cache is trimmed, else all."""
    page, pages = case["page"], -(-end // case["page"])
    if not case["trimmed"]:
        return list(range(pages))
    begin = max(0, first + 1 - case["window"])
    return [i for i in range(pages)
            if (i + 1) * page > begin or i * page < min(case["sinks"], end)]


def _tables(seed, held, max_pages):
    """Block tables that hold the given logical pages, over a pool of just the
    pages needed, in random order."""
    order = list(range(sum(len(h) for h in held)))
    random.Random(seed * 104729 + 5).shuffle(order)
    rows, at = [], 0
    for h in held:
        row = [-1] * max_pages
        for i in h:
            row[i] = order[at]
            at += 1
        rows.append(row)
    return rows, len(order)


def _attention_inputs(case, seed):
    g, d, page = _generator(seed), case["dim"], case["page"]
    if case["kind"] == "decode":
        lengths, queries = _lengths(case, seed), case["batch"]
        held = [_held(case, n - 1, n) for n in lengths]
        max_pages = -(-case["high"] // page)
    else:
        queries, end = case["rows"], case["start"] + case["rows"]
        lengths = list(range(case["start"] + 1, end + 1))
        held = [_held(case, case["start"], end)]
        max_pages = -(-end // page)
    table, pages = _tables(seed, held, max_pages)
    pool = (pages, case["kv_heads"], page, d)
    return dict(case=case, q=_normal(g, queries, case["heads"] * d), k=_normal(g, *pool),
                v=_normal(g, *pool), lengths=_i32(lengths), tables=_i32(table),
                active=_i32([case["active"]]), max_pages=max_pages,
                out=torch.zeros(queries, case["heads"] * d, dtype=F16, device="cuda"))


def _move_plan(case, seed):
    """(moves, tables, parents, remap, tail slots, tails): what the bookkeeping
    of a server has decided, as lists.  A move is (layer, source page,
    destination page, positions)."""
    rng = random.Random(seed * 15485863 + 3)
    layers, page, pages = case["layers"], case["page"], case["pages"]
    moves, tables = [], []
    if case["style"] == "fork":
        lengths = _spread(case["low"], case["high"], case["parents"])
        rng.shuffle(lengths)
        max_pages = -(-case["high"] // page)
        parents = [r for r in range(case["parents"]) for _ in range(case["children"])]
        slots = [(lengths[r] - 1) // page for r in parents]
        tails = []
        for layer in range(layers):
            order = list(range(pages))
            rng.shuffle(order)
            rows = []
            for n in lengths:
                row = [order.pop() for _ in range(-(-n // page))]
                rows.append(row + [-1] * (max_pages - len(row)))
            tables.append(rows)
            fresh = []
            for child, r in enumerate(parents):
                filled = lengths[r] - slots[child] * page
                fresh.append(order.pop())
                moves.append((layer, rows[r][slots[child]], fresh[-1], filled))
            tails.append(fresh)
        return moves, tables, parents, None, slots, tails
    live = max(1, int(pages * case["live"]))
    max_pages = -(-live // case["rows"])
    remap = []
    for layer in range(layers):
        used = rng.sample(range(pages), live)
        cells = used + [-1] * (case["rows"] * max_pages - live)
        tables.append([cells[r * max_pages:(r + 1) * max_pages] for r in range(case["rows"])])
        taken = set(used)
        holes = [p for p in range(live) if p not in taken]
        to = list(range(pages))
        for source in sorted(p for p in used if p >= live):
            to[source] = holes.pop()
            moves.append((layer, source, to[source], page))
        remap.append(to)
    if not moves:  # already packed: one page moves to a free place
        source, target = tables[0][0][0], pages - 1
        moves.append((0, source, target, page))
        remap[0][source] = target
    return moves, tables, None, remap, None, None


def _move_inputs(case, seed):
    g = _generator(seed)
    pools = (case["layers"], case["pages"], case["heads"], case["page"], case["dim"])
    keys, values = _normal(g, *pools), _normal(g, *pools)
    moves, tables, parents, remap, slots, tails = _move_plan(case, seed)
    state = dict(case=case, keys=keys, values=values, key_pools=list(keys),
                 value_pools=list(values), moves=_i32(moves), tables=_i32(tables), parents=None,
                 remap=None, slots=None, tails=None)
    for name, value in (("parents", parents), ("remap", remap), ("slots", slots),
                        ("tails", tails)):
        if value is not None:
            state[name] = _i32(value)
    rows = len(parents) if parents is not None else case["rows"]
    state["out"] = torch.zeros(case["layers"], rows, state["tables"].shape[2], dtype=torch.int32,
                               device="cuda")
    return state


def _score_inputs(case, seed):
    g, rows, vocab = _generator(seed), case["rows"], case["vocab"]
    logits = torch.randn(rows, vocab, generator=g, device="cuda") * 3.0
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    if case["masked"]:
        # the same tokens are forbidden in every row; a forbidden one is not chosen
        forbidden = torch.rand(vocab, generator=g, device="cuda") < case["masked"]
        forbidden[vocab // 2] = False
        logits.masked_fill_(forbidden, -math.inf)
        tokens = torch.where(forbidden[tokens.long()], vocab // 2, tokens).int()
    if case["type"] == "f16":
        logits = logits.to(F16)
    if case["padded"]:
        tokens[-1] = -1  # the last row of a prompt has no next token
    return dict(case=case, logits=logits, tokens=tokens)


def prepare(case, seed):
    if case["kind"] == "moves":
        return _move_inputs(case, seed)
    if case["kind"] == "score":
        state, rows, top = _score_inputs(case, seed), case["rows"], case["top"]
        state["out"] = [torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda"),
                        torch.zeros(rows, top, dtype=torch.int32, device="cuda"),
                        torch.zeros(rows, top, device="cuda")]
        if own:
            state["workspace"] = torch.zeros(
                max(1, _tmc().logprobs_workspace_bytes(rows, case["vocab"], top) // 4),
                device="cuda")
        return state
    state = _attention_inputs(case, seed)
    if own and case["kind"] == "decode":
        state["workspace"] = torch.zeros(
            max(1, _tmc().window_attention_workspace_bytes(
                case["batch"], case["heads"], case["kv_heads"], case["dim"],
                state["max_pages"] * case["page"], case["window"], case["sinks"]) // 4),
            device="cuda")
    return state


# ---------------------------------------------------------------- one pass
def _softmax(s):
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_decode(t):
    c = t["case"]
    n, window, sinks, page, dim = c["active"], c["window"], c["sinks"], c["page"], c["dim"]
    group = c["heads"] // c["kv_heads"]
    length = t["lengths"][:n, None].long()
    window, sinks = min(window, c["high"]), min(sinks, c["high"])
    first = torch.arange(sinks, device="cuda")[None, :].expand(n, -1)
    last = length - window + torch.arange(window, device="cuda")[None, :]
    position = torch.cat([first, last], 1)
    visible = torch.cat([first < length - window, last >= 0], 1)
    position = torch.where(visible, position, length - 1)
    pages = torch.gather(t["tables"][:n].long(), 1, position // page)
    k = t["k"][pages, :, position % page].float()  # [rows, positions, kv heads, dim]
    v = t["v"][pages, :, position % page].float()
    q = t["q"][:n].float().reshape(n, c["kv_heads"], group, dim)
    s = q @ k.permute(0, 2, 3, 1).contiguous() * (1.0 / math.sqrt(dim))
    p = _softmax(torch.where(visible[:, None, None, :], s, -math.inf))
    out = p @ v.permute(0, 2, 1, 3).contiguous()
    t["out"][:n] = out.reshape(n, -1).to(F16)
    return t["out"]


def _plain_chunk(t):
    c = t["case"]
    n, page, dim, kvh = c["active"], c["page"], c["dim"], c["kv_heads"]
    begin = max(0, c["start"] + 1 - c["window"])
    position = torch.cat([torch.arange(min(c["sinks"], begin), device="cuda"),
                          torch.arange(begin, c["start"] + n, device="cuda")])
    pages = t["tables"][0].long()[position // page]
    k = t["k"][pages, :, position % page].float().permute(1, 2, 0).contiguous()
    v = t["v"][pages, :, position % page].float().permute(1, 0, 2).contiguous()
    at = t["lengths"][:n, None].long() - 1
    visible = (position <= at) & ((position > at - c["window"]) | (position < c["sinks"]))
    q = t["q"][:n].float().reshape(n, kvh, c["heads"] // kvh, dim).permute(1, 2, 0, 3)
    s = q @ k[:, None] * (1.0 / math.sqrt(dim))  # [kv heads, group, rows, positions]
    out = _softmax(torch.where(visible, s, -math.inf)) @ v[:, None]
    t["out"][:n] = out.permute(2, 0, 1, 3).reshape(n, -1).to(F16)
    return t["out"]


def _plain_moves(t):
    c, moves = t["case"], t["moves"].long()
    slot = torch.arange(c["page"], device="cuda")
    for layer in range(c["layers"]):
        mine = moves[moves[:, 0] == layer]
        part = slot[None, :] < mine[:, 3:]
        for pool in (t["key_pools"][layer], t["value_pools"][layer]):
            pool[mine[:, 2]] = torch.where(part[:, None, :, None], pool[mine[:, 1]],
                                           pool[mine[:, 2]])
    tables = t["tables"]
    if t["parents"] is not None:
        tables = tables[:, t["parents"].long()]
    if t["remap"] is not None:
        flat = tables.reshape(c["layers"], -1)
        to = torch.gather(t["remap"], 1, flat.clamp(min=0).long())
        tables = torch.where(flat >= 0, to, flat).reshape(tables.shape)
    if t["slots"] is not None:
        here = torch.arange(tables.shape[2], device="cuda") == t["slots"][:, None]
        tables = torch.where(here, t["tails"][:, :, None], tables)
    t["out"].copy_(tables)
    return [t["out"], t["keys"], t["values"]]


def _plain_score(t):
    c = t["case"]
    x, vocab = t["logits"].float(), c["vocab"]
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    logprob, entropy, tokens, alternatives = t["out"]
    index = t["tokens"].clamp(min=0).long()[:, None]
    given = torch.gather(x, 1, index) - top - log_total
    logprob.copy_(torch.where(t["tokens"] >= 0, given[:, 0], logprob))
    mean = torch.where(e > 0, e * (x - top), 0.0).sum(-1, keepdim=True) / total
    entropy.copy_((log_total - mean)[:, 0])
    if c["top"]:
        # the greatest first and the lower index first among equals, as one key
        bits = x.view(torch.int32) if x.is_contiguous() else x.contiguous().view(torch.int32)
        order = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long()
        key = order * 2 ** 20 + (2 ** 20 - 1 - torch.arange(vocab, device="cuda"))
        best = torch.topk(key, c["top"], -1).values
        which = 2 ** 20 - 1 - best % 2 ** 20
        tokens.copy_(which)
        alternatives.copy_(torch.gather(x, 1, which) - top - log_total)
    return t["out"]


def run(state):
    c = state["case"]
    if not own:
        return {"decode": _plain_decode, "chunk": _plain_chunk, "moves": _plain_moves,
                "score": _plain_score}[c["kind"]](state)
    tmc = _tmc()
    if c["kind"] == "moves":
        tmc.move_pages(state["key_pools"], state["value_pools"], state["moves"], c["heads"],
                       c["page"], c["dim"])
        tmc.rebuild_tables(state["tables"], state["out"], c["pages"], parents=state["parents"],
                           remap=state["remap"], tail_slots=state["slots"], tails=state["tails"])
        return [state["out"], state["keys"], state["values"]]
    if c["kind"] == "score":
        logprob, entropy, tokens, alternatives = state["out"]
        tmc.logprobs(state["logits"], state["tokens"], logprob, entropy, tokens, alternatives,
                     state["workspace"])
        return state["out"]
    head_stride = c["page"] * c["dim"]
    geometry = (c["heads"], c["kv_heads"], c["dim"], c["page"], state["max_pages"],
                c["kv_heads"] * head_stride, head_stride, c["window"], c["sinks"])
    if c["kind"] == "decode":
        tmc.window_decode_attention(state["q"], state["k"], state["v"], state["lengths"],
                                    state["tables"], state["active"], state["out"], c["batch"],
                                    *geometry, workspace=state["workspace"])
    else:
        tmc.window_prefill_attention(state["q"], state["k"], state["v"], state["lengths"],
                                     state["tables"], None, state["active"], state["out"],
                                     c["rows"], *geometry)
    return state["out"]


# ---------------------------------------------------------------- bounds
def _visible(length, window, sinks):
    begin = max(0, length - window)
    return length - begin + min(sinks, begin)


def work(case):
    """Bytes read and written once and operations of one pass."""
    kind = case["kind"]
    if kind == "moves":
        row = 2 * case["heads"] * case["dim"]
        if case["style"] == "fork":
            lengths = _spread(case["low"], case["high"], case["parents"])
            slots = -(-case["high"] // case["page"])
            # a tail is read once for all its children
            tails = sum(n - (n - 1) // case["page"] * case["page"] for n in lengths)
            positions = tails * (1 + case["children"])
            cells = case["parents"] * slots * (1 + case["children"])
            moved = case["parents"] * case["children"]
        else:
            live = max(1, int(case["pages"] * case["live"]))
            # the expected number of live pages that lie behind the packed ones
            moved = live * (1.0 - live / case["pages"])
            positions = 2 * moved * case["page"]
            cells = 2 * live + case["pages"]
        return dict(bytes=case["layers"] * (2 * positions * row + 4 * cells + 16 * moved),
                    flops=0)
    if kind == "score":
        size = 4 if case["type"] == "f32" else 2
        count = case["rows"] * case["vocab"]
        return dict(bytes=size * count + case["rows"] * (12 + 8 * case["top"]), flops=5.0 * count)
    heads, kvh, d, window, sinks = (case[n] for n in ("heads", "kv_heads", "dim", "window",
                                                      "sinks"))
    if kind == "decode":
        # the active rows are a random part of the batch: their expected share
        lengths = _spread(case["low"], case["high"], case["batch"])
        seen = (sum(_visible(n, window, sinks) for n in lengths) * case["active"]
                / case["batch"])
        return dict(bytes=seen * kvh * d * 4 + 4 * case["active"] * heads * d,
                    flops=seen * heads * d * 4.0)
    n, start = case["active"], case["start"]
    pairs = sum(_visible(start + r + 1, window, sinks) for r in range(n))
    begin = max(0, start + 1 - window)
    keys = start + n - begin + min(sinks, begin)
    return dict(bytes=keys * kvh * d * 4 + 4 * n * heads * d, flops=pairs * heads * d * 4.0)


# ---------------------------------------------------------------- 64 bits
def _attend64(q, k, v, see):
    """q [rows, heads, dim] over k, v [positions, kv heads, dim] where see
    [rows, positions]."""
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    group = q.shape[1] // k.shape[1]
    for head in range(q.shape[1]):
        kh = k[:, head // group].double()
        s = (q[:, head].double() @ kh.t().contiguous()) / math.sqrt(q.shape[2])
        s[~see] = -math.inf
        w = torch.softmax(s, -1)
        out[:, head] = w @ v[:, head // group].double()
    return out


def _sequence(pool, row, wanted, page):
    """The wanted positions of one block-table row: [positions, kv heads, dim]."""
    flat = pool.permute(0, 2, 1, 3).reshape(-1, pool.shape[1], pool.shape[3])
    index = [row[p // page] * page + p % page for p in wanted]
    return flat[torch.tensor(index, device="cuda")]


def _exact_attention(case, seed):
    t = _attention_inputs(case, seed)
    tables, lengths = t["tables"].tolist(), t["lengths"].tolist()
    heads, dim = case["heads"], case["dim"]
    out = torch.zeros(t["out"].shape, dtype=torch.float64, device="cuda")
    q = t["q"].reshape(-1, heads, dim)
    if case["kind"] == "decode":
        groups = [([r], tables[r]) for r in range(case["active"])]
    else:
        groups = [(list(range(case["active"])), tables[0])]
    for rows, row in groups:
        last = [lengths[r] - 1 for r in rows]
        low = max(0, last[0] + 1 - case["window"])
        wanted = [p for p in range(last[-1] + 1) if p >= low or p < case["sinks"]]
        k, v = (_sequence(t[n], row, wanted, case["page"]) for n in ("k", "v"))
        p, at = torch.tensor(wanted, device="cuda"), torch.tensor(last, device="cuda")[:, None]
        see = (p[None, :] <= at) & ~((p[None, :] <= at - case["window"])
                                     & (p[None, :] >= case["sinks"]))
        out[rows] = _attend64(q[rows], k, v, see).reshape(len(rows), -1)
    return out


def _exact_moves(case, seed):
    t = _move_inputs(case, seed)
    moves, tables, parents, remap, slots, tails = _move_plan(case, seed)
    rows = range(case["rows"]) if parents is None else range(len(parents))
    out = []
    for layer, table in enumerate(tables):
        new = []
        for r in rows:
            row = list(table[r if parents is None else parents[r]])
            if remap is not None:
                row = [p if p < 0 else remap[layer][p] for p in row]
            if slots is not None:
                row[slots[r]] = tails[layer][r]
            new.append(row)
        out.append(new)
    for pools in (t["keys"], t["values"]):
        for layer, pool in enumerate(pools):
            mine = [m[1:] for m in moves if m[0] == layer]
            for filled in {m[2] for m in mine}:
                source, target = (torch.tensor([m[i] for m in mine if m[2] == filled],
                                               device="cuda") for i in (0, 1))
                pool[target, :, :filled] = pool[source, :, :filled]
    return [_i32(out), t["keys"].double(), t["values"].double()]


def _exact_score(case, seed):
    t = _score_inputs(case, seed)
    x = t["logits"].double()
    logp = x - torch.logsumexp(x, -1, keepdim=True)
    p = torch.exp(logp)
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    given = logp.gather(1, t["tokens"].clamp(min=0).long()[:, None])[:, 0]
    given = torch.where(t["tokens"] >= 0, given, 0.0)
    which = torch.sort(x, stable=True, dim=-1, descending=True).indices[:, :case["top"]]
    return [given, entropy, which.int(), logp.gather(1, which)]


def exact(case, seed):
    if case["kind"] == "moves":
        return _exact_moves(case, seed)
    if case["kind"] == "score":
        return _exact_score(case, seed)
    return _exact_attention(case, seed)
