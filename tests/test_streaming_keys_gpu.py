"""The streaming-generation kernels through the runtime's keys: bindings,
refusals, and a sequence of them that replays with the results of the direct
calls (which their own tests hold against 64 bits)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "GPU tests need a GPU"
    return t


@pytest.mark.parametrize("key,text", [
    ("window_attention?max_batch=2&q_heads=8&head_dim=128&page_size=16&max_pages=4", "window"),
    ("window_attention?max_batch=2&q_heads=8&head_dim=128&page_size=16&max_pages=4&window=8"
     "&dtype=f32", "f16"),
    ("window_attention?max_batch=2&q_heads=8&head_dim=128&page_size=16&max_pages=4&window=8"
     "&out_layout=tiled", "out_layout"),
    ("window_prefill_attention?rows=4&q_heads=8&head_dim=128&page_size=16&max_pages=4", "window"),
    ("window_prefill_attention?rows=4&q_heads=8&head_dim=128&page_size=16&max_pages=4&window=8"
     "&tables=-1", "tables"),
    ("move_pages?heads=8&head_dim=128&page_size=16", "moves"),
    ("move_pages?moves=4&heads=8&head_dim=128&page_size=16&pools=16", "pools"),
    ("rebuild_tables?rows=4&max_pages=8", "pool_pages"),
    ("rebuild_tables?rows=4&table_rows=2&max_pages=8&pool_pages=16", "parents"),
    ("logprobs?rows=4", "vocab"), ("logprobs?rows=4&vocab=100&dtype=bf16", "dtype"),
    ("logprobs?rows=4&vocab=100&top=65", "top"), ("logprobs?rows=4&vocab=10&top=11", "top")])
def test_keys_refuse(tmc, torch, key, text):
    with pytest.raises(RuntimeError, match=text):
        tmc.Runtime().resolve(key)


def test_keys_check_their_buffers(tmc, torch):
    rt = tmc.Runtime()
    key = rt.resolve("logprobs?rows=4&vocab=100")
    logits = rt.create_buffer(4 * 100, tmc.F32)
    tokens, short = rt.create_buffer(4, tmc.I32), rt.create_buffer(3, tmc.F32)
    with pytest.raises(RuntimeError):
        rt.prepare(key, [logits, tokens], [short, rt.create_buffer(4, tmc.F32)])


@pytest.mark.parametrize("qh,kvh,d,tables,packed", [(8, 2, 128, 0, False), (4, 4, 64, 3, True)])
def test_a_sequence_of_them_replays(tmc, torch, qh, kvh, d, tables, packed):
    page, max_pages, batch, window, sinks, pages, vocab, top = 16, 6, 3, 40, 5, 32, 5000, 4
    g = torch.Generator(device="cuda")
    g.manual_seed(qh * d)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(torch.float16)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    k, v = normal(pages, kvh, page, d), normal(pages, kvh, page, d)
    parents = ints([1, 1, 0])
    old = torch.randperm(pages - 4, generator=g, device="cuda")[:2 * max_pages].to(torch.int32)
    slots, tails = ints([3, -1, -1]), ints([pages - 1, 0, 0])
    moves = ints([(0, int(old[max_pages + 3]), pages - 1, 9)])
    q, valid, active = normal(batch, qh * d), ints([50, 49, 3 * page]), ints([batch])
    rows = 7
    chunk_q, chunk_valid, chunk_active = normal(rows, qh * d), ints([43, 44, 45, 46, 47, 48, 49]), ints([rows])
    row_table = ints([0, 0, 1, 1, 1, 2, 2])
    logits = torch.randn(batch, vocab, generator=g, device="cuda")
    tokens = ints([7, -1, vocab - 1])

    def outputs():
        wide = tmc.packed_activation_elements(batch, qh * d) if packed else batch * qh * d
        return dict(tables=torch.full((1, batch, max_pages), -7, dtype=torch.int32, device="cuda"),
                    out=torch.full((wide,), 3.0, dtype=torch.float16, device="cuda"),
                    chunk=torch.full((rows, qh * d), 3.0, dtype=torch.float16, device="cuda"),
                    logprob=torch.full((batch,), 9.0, device="cuda"),
                    entropy=torch.full((batch,), 9.0, device="cuda"),
                    top=torch.full((batch, top), 9, dtype=torch.int32, device="cuda"),
                    best=torch.full((batch, top), 9.0, device="cuda"))

    # the direct calls, on pools of their own
    want = outputs()
    kw, vw = k.clone(), v.clone()
    tmc.move_pages([kw], [vw], moves, kvh, page, d)
    tmc.rebuild_tables(old.reshape(1, 2, max_pages), want["tables"], pages, parents=parents,
                       tail_slots=slots, tails=tails)
    geometry = (qh, kvh, d, page, max_pages, kvh * page * d, page * d, window, sinks)
    ws = torch.zeros(tmc.window_attention_workspace_bytes(batch, qh, kvh, d, page * max_pages,
                                                          window, sinks) // 4 + 1, device="cuda")
    tmc.window_decode_attention(q, kw, vw, valid, want["tables"], active, want["out"], batch,
                                *geometry, workspace=ws, layout=tmc.Y_PACKED if packed else 0)
    some = want["tables"][0] if tables else want["tables"][0, :1]
    tmc.window_prefill_attention(chunk_q, kw, vw, chunk_valid, some, row_table if tables else None,
                                 chunk_active, want["chunk"], rows, *geometry)
    tmc.logprobs(logits, tokens, want["logprob"], want["entropy"], want["top"], want["best"],
                 torch.zeros(tmc.logprobs_workspace_bytes(batch, vocab, top) // 4 + 1,
                             device="cuda"))
    torch.cuda.synchronize()

    rt = tmc.Runtime()
    got = outputs()
    wrapped = []

    def bind(t):
        wrapped.append(rt.wrap(t))
        return wrapped[-1]

    kb, vb, tb = bind(k), bind(v), bind(got["tables"])
    shape = f"q_heads={qh}&kv_heads={kvh}&head_dim={d}&page_size={page}&max_pages={max_pages}"
    shape += f"&window={window}&sinks={sinks}"
    steps = [
        rt.prepare(rt.resolve(f"move_pages?moves=1&heads={kvh}&head_dim={d}&page_size={page}"),
                   [bind(moves)], [kb, vb]),
        rt.prepare(rt.resolve(f"rebuild_tables?rows={batch}&table_rows=2&max_pages={max_pages}"
                              f"&pool_pages={pages}&parents=1&tails=1"),
                   [bind(old), bind(parents), bind(slots), bind(tails)], [tb]),
        rt.prepare(rt.resolve(f"window_attention?max_batch={batch}&{shape}"
                              + ("&out_layout=packed" if packed else "")),
                   [bind(q), kb, vb, bind(valid), tb, bind(active)], [bind(got["out"])]),
        rt.prepare(rt.resolve(f"window_prefill_attention?rows={rows}&{shape}"
                              + (f"&tables={tables}" if tables else "")),
                   [bind(chunk_q), kb, vb, bind(chunk_valid), tb]
                   + ([bind(row_table)] if tables else []) + [bind(chunk_active)],
                   [bind(got["chunk"])]),
        rt.prepare(rt.resolve(f"logprobs?rows={batch}&vocab={vocab}&top={top}"),
                   [bind(logits), bind(tokens)],
                   [bind(got[n]) for n in ("logprob", "entropy", "top", "best")])]
    sequence = rt.sequence(steps)
    for _ in range(4):
        fresh = outputs()
        for name in ("out", "chunk", "logprob", "entropy", "top", "best"):
            got[name].copy_(fresh[name])
        torch.cuda.synchronize()
        sequence.run()
        torch.cuda.synchronize()
        assert torch.equal(k, kw) and torch.equal(v, vw)
        for name, t in want.items():
            assert torch.equal(got[name], t), name
    assert float(got["logprob"][1]) == 9.0  # token -1: left as it was
    assert np.isfinite(got["logprob"][0].item())
