"""Refusals of the streaming-generation entry points, without a device: every
bad argument fails before any device work, and the host check of page moves."""
import ctypes as C

import pytest

P = C.c_void_p(4096)  # a 16-byte aligned address that no refused call reads
ODD = C.c_void_p(4104)


def decode(lib, q=P, k=P, v=P, valid=P, tables=P, out=P, dtype=0, batch=2, qh=8, kvh=2, d=128,
           page=16, pages=4, pool=8, page_stride=2 * 16 * 128, head_stride=16 * 128, window=8,
           sinks=2, workspace=P, ws_bytes=1 << 40, layout=0):
    return lib.tmc_window_decode_attention(q, k, v, valid, tables, None, out, dtype, batch, qh, kvh,
                                           d, page, pages, pool, page_stride, head_stride, window,
                                           sinks, workspace, ws_bytes, layout, None)


@pytest.mark.parametrize("change,text", [
    (dict(q=None), "null"), (dict(tables=None), "null"), (dict(out=None), "null"),
    (dict(dtype=1), "fp16"), (dict(d=12), "head_dim"), (dict(d=264), "head_dim"),
    (dict(d=0), "head_dim"), (dict(qh=7), "heads"), (dict(batch=0), "rows"),
    (dict(batch=65536), "max_batch"), (dict(page=0), "geometry"), (dict(pages=1 << 28), "geometry"),
    (dict(pool=0), "geometry"), (dict(head_stride=16 * 128 - 8), "strides"),
    (dict(page_stride=2 * 16 * 128 + 4), "strides"), (dict(page_stride=16 * 128), "strides"),
    (dict(k=ODD), "aligned"), (dict(out=ODD), "aligned"), (dict(window=0), "window"),
    (dict(window=-1), "window"), (dict(sinks=-1), "sinks"), (dict(layout=1), "layout"),
])
def test_window_decode_refuses(tmc, change, text):
    assert decode(tmc.lib(), **change) != 0
    assert text in tmc.last_error()


def test_window_decode_needs_its_workspace(tmc):
    need = tmc.window_attention_workspace_bytes(4, 32, 8, 128, 4096, 2048, 4)
    if need:
        for ws, size in ((P, need - 1), (None, need)):
            assert decode(tmc.lib(), batch=4, qh=32, kvh=8, pages=256, page_stride=8 * 16 * 128,
                          window=2048, sinks=4, workspace=ws, ws_bytes=size) != 0
            assert "workspace" in tmc.last_error()
    assert tmc.window_attention_workspace_bytes(0, 32, 8, 128, 4096, 2048, 4) == 0
    assert tmc.window_attention_workspace_bytes(4, 33, 8, 128, 4096, 2048, 4) == 0


def chunk(lib, tables=P, row_table=None, table_rows=1, active=P, d=128, window=8, rows=4):
    return lib.tmc_window_prefill_attention_f16(P, P, P, P, tables, row_table, table_rows, active,
                                                P, rows, 8, 2, d, 16, 4, 8, 2 * 16 * d, 16 * d,
                                                window, 2, None)


@pytest.mark.parametrize("change,text", [
    (dict(active=None), "active"), (dict(table_rows=2), "table_rows"),
    (dict(row_table=P, table_rows=0), "table_rows"), (dict(d=20), "head_dim"),
    (dict(window=0), "window"), (dict(rows=0), "rows"), (dict(rows=1 << 24), "rows"),
    (dict(tables=None), "null")])
def test_window_chunk_refuses(tmc, change, text):
    assert chunk(tmc.lib(), **change) != 0
    assert text in tmc.last_error()


def move(lib, keys=(P,), values=(P,), moves=P, count=1, dtype=0, pages=8, heads=2, page=16, d=128,
         page_stride=2 * 16 * 128, head_stride=16 * 128):
    k = (C.c_void_p * len(keys))(*[x.value if x else None for x in keys])
    v = (C.c_void_p * len(values))(*[x.value if x else None for x in values])
    return lib.tmc_move_pages(k, v, len(keys), moves, count, dtype, pages, heads, page, d,
                              page_stride, head_stride, None)


@pytest.mark.parametrize("change,text", [
    (dict(moves=None), "null"), (dict(keys=(None,)), "null pool"), (dict(dtype=3), "dtype"),
    (dict(count=-1), "shape"), (dict(pages=0), "shape"), (dict(heads=0), "shape"),
    (dict(page=0), "shape"), (dict(d=0), "shape"), (dict(head_stride=8), "stride"),
    (dict(page_stride=16 * 128), "stride"), (dict(moves=ODD), "16-byte"),
    (dict(keys=(C.c_void_p(4097),)), "aligned")])
def test_move_pages_refuses(tmc, change, text):
    assert move(tmc.lib(), **change) != 0
    assert text in tmc.last_error()


def test_no_moves_are_nothing(tmc):
    assert move(tmc.lib(), count=0) == 0


@pytest.mark.parametrize("moves,text", [
    ([(0, 1, 2, 16), (0, 3, 2, 4)], "another move writes"),
    ([(0, 1, 2, 16), (0, 2, 3, 4)], "both read and written"),
    ([(0, 5, 5, 3)], "both read and written"),
    ([(0, 8, 2, 16)], "does not exist"), ([(0, -1, 2, 16)], "does not exist"),
    ([(0, 1, 8, 16)], "does not exist"), ([(2, 1, 2, 16)], "does not exist"),
    ([(0, 1, 2, 0)], "positions"), ([(0, 1, 2, 17)], "positions")])
def test_page_moves_are_checked(tmc, moves, text):
    with pytest.raises(RuntimeError, match=text):
        tmc.page_moves(moves, 2, 8, 16)


def test_good_page_moves_pass(tmc):
    flat = (C.c_int32 * 16)(*[0, 1, 2, 16, 0, 1, 3, 4, 1, 2, 1, 5, 1, 2, 3, 1])
    assert tmc.lib().tmc_check_page_moves(flat, 4, 2, 8, 16) == 0
    assert tmc.lib().tmc_check_page_moves(None, 0, 2, 8, 16) == 0


def rebuild(lib, tables=4096, parents=None, remap=None, slots=None, tails=None, out=1 << 20,
            layers=2, table_rows=4, rows=4, pages=8, pool=16):
    p = lambda x: None if x is None else C.c_void_p(x)  # noqa: E731
    return lib.tmc_rebuild_tables(p(tables), p(parents), p(remap), p(slots), p(tails), p(out),
                                  layers, table_rows, rows, pages, pool, None)


@pytest.mark.parametrize("change,text", [
    (dict(tables=None), "null"), (dict(out=None), "null"), (dict(slots=4096), "go together"),
    (dict(tails=4096), "go together"), (dict(rows=5), "without parents"), (dict(rows=0), "shape"),
    (dict(pages=1 << 30), "shape"), (dict(layers=0), "shape"), (dict(pool=0), "shape"),
    (dict(out=4100), "overlap"), (dict(parents=64, out=4096), "overlap")])
def test_rebuild_tables_refuses(tmc, change, text):
    assert rebuild(tmc.lib(), **change) != 0
    assert text in tmc.last_error()


def score(lib, logits=P, dtype=1, stride=1000, tokens=P, logprob=P, entropy=P, tops=P, values=P,
          rows=4, vocab=1000, top=5, workspace=P, ws_bytes=1 << 40):
    return lib.tmc_logprobs(logits, dtype, stride, tokens, logprob, entropy, tops, values, rows,
                            vocab, top, workspace, ws_bytes, None)


@pytest.mark.parametrize("change,text", [
    (dict(logits=None), "null"), (dict(dtype=2), "f32 or f16"), (dict(stride=999), "shape"),
    (dict(rows=0), "shape"), (dict(vocab=0), "shape"), (dict(top=65), "top"),
    (dict(top=-1), "top"), (dict(vocab=3, stride=3), "top"), (dict(tokens=None), "go together"),
    (dict(logprob=None), "go together"), (dict(tops=None), "alternatives"),
    (dict(logits=C.c_void_p(4098)), "aligned")])
def test_logprobs_refuses(tmc, change, text):
    assert score(tmc.lib(), **change) != 0
    assert text in tmc.last_error()


def test_logprobs_needs_its_workspace(tmc):
    need = tmc.logprobs_workspace_bytes(16, 32000, 20)
    if need:
        for ws, size in ((P, need - 1), (None, need)):
            assert score(tmc.lib(), rows=16, vocab=32000, stride=32000, top=20, workspace=ws,
                         ws_bytes=size) != 0
            assert "workspace" in tmc.last_error()
    assert tmc.logprobs_workspace_bytes(0, 32000, 20) == 0
