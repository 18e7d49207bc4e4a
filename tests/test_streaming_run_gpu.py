"""The streaming operators as a server uses them together: a prompt enters the
cache in chunks under a window, is forked into several continuations that share
its full pages, decodes them step by step with their pages given back as the
window passes and the pool packed in between, and every step's logits give the
tokens their log probabilities.  Each row is compared with a plain 64-bit model
of its own sequence (attention over its own keys and values), so a page that
is shared, moved or freed wrongly shows."""
import math

import pytest

from tests.test_window_gpu import attend64, visible

pytestmark = pytest.mark.gpu


def test_prompt_fork_decode_compact_score(tmc):
    import torch
    layers, qh, kvh, d, page, window, sinks = 2, 8, 2, 128, 16, 70, 4
    cap_pages, pages, vocab, children = 12, 64, 1003, 3
    capacity = cap_pages * page
    prompt, steps, chunk = 101, 50, 37
    g = torch.Generator(device="cuda")
    g.manual_seed(41)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.float16)  # noqa: E731
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    keys = [torch.full((pages, kvh, page, d), math.nan, dtype=torch.float16, device="cuda")
            for _ in range(layers)]
    values = [t.clone() for t in keys]
    width, kv = qh * d, kvh * d
    cos = torch.ones(capacity, d // 2, device="cuda")   # the identity rotation: the cache
    sin = torch.zeros(capacity, d // 2, device="cuda")  # holds the keys as they are given
    strides = (kvh * page * d, page * d)
    free = list(range(pages))[::-1]
    shared = {}  # page -> number of rows that hold it (the same in every layer)

    def take():
        shared[free[-1]] = 1
        return free.pop()

    def give(p):
        shared[p] -= 1
        if not shared[p]:
            del shared[p]
            free.append(p)

    # ---- the prompt, in chunks
    table = [take() for _ in range(-(-prompt // page))]
    table += [-1] * (cap_pages - len(table))
    history = [[[], []] for _ in range(layers)]  # per layer: rows' k and v so far
    for start in range(0, prompt, chunk):
        rows = min(chunk, prompt - start)
        valid = i32(list(range(start + 1, start + rows + 1)))
        for layer in range(layers):
            qkv = rand(rows, width + 2 * kv)
            q = torch.zeros(rows, width, dtype=torch.float16, device="cuda")
            tmc.prefill_rope_append(qkv, cos, sin, valid, i32(table), i32([rows]), q, keys[layer],
                                    values[layer], rows, qh, kvh, d, capacity, page, cap_pages)
            out = torch.zeros_like(q)
            tmc.window_prefill_attention(q, keys[layer], values[layer], valid, i32([table]), None,
                                         i32([rows]), out, rows, qh, kvh, d, page, cap_pages,
                                         *strides, window, sinks)
            history[layer][0].append(qkv[:, width:width + kv].reshape(rows, kvh, d))
            history[layer][1].append(qkv[:, width + kv:].reshape(rows, kvh, d))
            kk, vv = (torch.cat(h) for h in history[layer])
            for r in (0, rows // 2, rows - 1):
                see = torch.tensor(visible(start + r + 1, window, sinks), device="cuda")
                o, tol = attend64(torch, qkv[r, :width].reshape(qh, d), kk[see], vv[see])
                assert ((out[r].double().reshape(qh, d) - o).abs() <= tol).all()

    # ---- fork: full pages shared, the partly filled one copied
    slot, filled = (prompt - 1) // page, prompt - (prompt - 1) // page * page
    assert 0 < filled < page
    tails = [table[slot]] + [take() for _ in range(children - 1)]
    moves = [(layer, table[slot], t, filled) for layer in range(layers) for t in tails[1:]]
    tmc.move_pages(keys, values, tmc.page_moves(moves, layers, pages, page), kvh, page, d)
    for p in table[:slot]:
        shared[p] += children - 1
    tables = torch.zeros(layers, children, cap_pages, dtype=torch.int32, device="cuda")
    tmc.rebuild_tables(i32([[table]] * layers), tables, pages, parents=i32([0] * children),
                       tail_slots=i32([slot] * children), tails=i32([tails] * layers))
    rows_now = [table[:slot] + [t] + [-1] * (cap_pages - slot - 1) for t in tails]
    assert tables.tolist() == [rows_now] * layers
    sequences = [[[torch.cat(h)] for h in history[layer] for _ in range(children)]
                 for layer in range(layers)]  # [layer][k rows of each child, then v]
    ws = torch.zeros(max(1, tmc.window_attention_workspace_bytes(children, qh, kvh, d, capacity,
                                                                 window, sinks) // 4), device="cuda")
    lm_head = rand(vocab, width)
    score_ws = torch.zeros(max(1, tmc.logprobs_workspace_bytes(children, vocab, 3) // 4), device="cuda")
    totals = torch.zeros(children, device="cuda")
    totals64 = torch.zeros(children, dtype=torch.float64, device="cuda")
    for step in range(steps):
        n = prompt + step + 1
        for r in range(children):
            at = (n - 1) // page
            if rows_now[r][at] < 0:
                rows_now[r][at] = take()
            for i in range(cap_pages):  # pages that the window has passed
                if rows_now[r][i] >= 0 and i * page >= sinks and (i + 1) * page <= n - window:
                    give(rows_now[r][i])
                    rows_now[r][i] = -1
        tables = i32([rows_now] * layers)
        valid, active = i32([n] * children), i32([children])
        for layer in range(layers):
            qkv = rand(children, width + 2 * kv)
            q = torch.zeros(children, width, dtype=torch.float16, device="cuda")
            tmc.decode_rope_append(qkv, cos, sin, valid, tables[layer], active, q, keys[layer],
                                   values[layer], children, qh, kvh, d, capacity, page, cap_pages)
            out = torch.zeros_like(q)
            tmc.window_decode_attention(q, keys[layer], values[layer], valid,
                                        tables[layer].contiguous(), active, out, children, qh, kvh,
                                        d, page, cap_pages, *strides, window, sinks, ws)
            for r in range(children):
                seq = sequences[layer][r], sequences[layer][children + r]
                seq[0].append(qkv[r:r + 1, width:width + kv].reshape(1, kvh, d))
                seq[1].append(qkv[r:r + 1, width + kv:].reshape(1, kvh, d))
                kk, vv = (torch.cat(s) for s in seq)
                see = torch.tensor(visible(n, window, sinks), device="cuda")
                o, tol = attend64(torch, qkv[r, :width].reshape(qh, d), kk[see], vv[see])
                assert ((out[r].double().reshape(qh, d) - o).abs() <= tol).all(), (step, layer, r)
        # the last layer's rows stand for the hidden state; greedy tokens with alternatives
        logits = torch.zeros(children, vocab, device="cuda")
        tmc.gemv(out, lm_head, logits)
        tokens = torch.zeros(children, dtype=torch.int32, device="cuda")
        tmc.argmax(logits, tokens)
        lp, entropy = torch.zeros(children, device="cuda"), torch.zeros(children, device="cuda")
        top = torch.zeros(children, 3, dtype=torch.int32, device="cuda")
        top_lp = torch.zeros(children, 3, device="cuda")
        tmc.logprobs(logits, tokens, lp, entropy, top, top_lp, score_ws)
        assert torch.equal(top[:, 0], tokens) and torch.equal(top_lp[:, 0], lp)
        totals += lp
        totals64 += torch.log_softmax(logits.double(), -1).amax(-1)
        if step == steps // 2:  # compact: live pages to the front, the sources spoiled
            live = sorted({p for row in rows_now for p in row if p >= 0})
            holes = [p for p in range(len(live)) if p not in live]
            to = list(range(pages))
            for p in live:
                if p >= len(live):
                    to[p] = holes.pop()
            moved = [(layer, p, to[p], page) for layer in range(layers) for p in live if to[p] != p]
            assert moved
            tmc.move_pages(keys, values, tmc.page_moves(moved, layers, pages, page), kvh, page, d)
            packed = torch.zeros_like(tables)
            tmc.rebuild_tables(tables, packed, pages, remap=i32([to] * layers))
            rows_now = packed[0].tolist()
            for layer in range(layers):
                keys[layer][len(live):], values[layer][len(live):] = math.nan, math.nan
            shared = {to[p]: c for p, c in shared.items()}
            assert sorted(shared) == list(range(len(live)))
            free = list(range(len(live), pages))[::-1]
    assert ((totals.double() - totals64).abs() < 1e-3).all()
    # what is held at the end is what the window and the sinks need, the sinks' page shared
    assert len(shared) <= 1 + children * (window // page + 2)
