"""Refusals of the speculative-decoding entry points, without a device: every bad
argument fails before any device work."""
import ctypes as C

import pytest

P = C.c_void_p(4096)  # a 16-byte aligned address that no refused call reads
ODD = C.c_void_p(4104)
HUGE = 1 << 40


def layout(lib, parents=P, masks=P, depths=P, batch=2, nodes=8):
    return lib.tmc_tree_layout(parents, None, masks, depths, batch, nodes, None)


@pytest.mark.parametrize("change,text", [
    (dict(parents=None), "null"), (dict(masks=None), "null"), (dict(depths=None), "null"),
    (dict(batch=0), "batch"), (dict(batch=65536), "batch"), (dict(nodes=0), "nodes"),
    (dict(nodes=257), "nodes"), (dict(nodes=-1), "nodes")])
def test_layout_refuses(tmc, change, text):
    assert layout(tmc.lib(), **change) != 0
    assert text in tmc.last_error()


def append(lib, qkv=P, cosine=P, sine=P, positions=64, cached=P, depths=P, tables=P, q=P, k=P, v=P,
           dtype=0, batch=2, nodes=8, qh=8, kvh=2, d=128, page=16, pages=4, pool=8):
    return lib.tmc_tree_rope_append(qkv, cosine, sine, positions, cached, depths, None, tables, None,
                                    q, k, v, dtype, batch, nodes, qh, kvh, d, page, pages, pool, None)


@pytest.mark.parametrize("change,text", [
    *[({n: None}, "null") for n in ("qkv", "cosine", "sine", "cached", "depths", "tables", "q", "k",
                                    "v")],
    (dict(dtype=2), "dtype"), (dict(dtype=3), "dtype"), (dict(batch=0), "batch"),
    (dict(nodes=300), "nodes"), (dict(qh=7), "heads"), (dict(kvh=0), "heads"), (dict(d=7), "heads"),
    (dict(d=1026), "heads"), (dict(positions=0), "heads"), (dict(page=0), "geometry"),
    (dict(pages=1 << 28), "geometry"), (dict(pool=0), "geometry"), (dict(pool=1 << 31), "geometry"),
    (dict(batch=65535, nodes=256, qh=64, kvh=8, d=256), "too many"),
    (dict(qkv=C.c_void_p(4098)), "aligned"), (dict(dtype=1, v=C.c_void_p(4100)), "aligned")])
def test_append_refuses(tmc, change, text):
    assert append(tmc.lib(), **change) != 0
    assert text in tmc.last_error()


def attend(lib, q=P, k=P, v=P, cached=P, masks=P, tables=P, out=P, dtype=0, batch=2, nodes=8, qh=8,
           kvh=2, d=128, page=16, pages=4, pool=8, page_stride=2 * 16 * 128, head_stride=16 * 128,
           workspace=P, ws_bytes=HUGE):
    return lib.tmc_tree_attention(q, k, v, cached, masks, None, tables, None, out, dtype, batch,
                                  nodes, qh, kvh, d, page, pages, pool, page_stride, head_stride,
                                  workspace, ws_bytes, None)


@pytest.mark.parametrize("change,text", [
    *[({n: None}, "null") for n in ("q", "k", "v", "cached", "masks", "tables", "out")],
    (dict(dtype=1), "fp16"), (dict(dtype=2), "fp16"), (dict(d=12), "head_dim"),
    (dict(d=264), "head_dim"), (dict(d=0), "head_dim"), (dict(qh=7), "heads"), (dict(kvh=0), "heads"),
    (dict(batch=0), "batch"), (dict(batch=65536), "batch"), (dict(nodes=0), "nodes"),
    (dict(nodes=257), "nodes"), (dict(page=0), "geometry"), (dict(pages=1 << 28), "geometry"),
    (dict(pool=0), "geometry"), (dict(head_stride=16 * 128 - 8), "strides"),
    (dict(page_stride=2 * 16 * 128 + 4), "strides"), (dict(page_stride=16 * 128), "strides"),
    (dict(q=ODD), "aligned"), (dict(k=ODD), "aligned"), (dict(out=ODD), "aligned")])
def test_attention_refuses(tmc, change, text):
    assert attend(tmc.lib(), **change) != 0
    assert text in tmc.last_error()


def test_attention_needs_its_workspace(tmc):
    need = tmc.tree_attention_workspace_bytes(1, 8, 32, 8, 128, 16 * 1000)
    if need:
        for ws, size in ((P, need - 1), (None, need), (ODD, need)):
            assert attend(tmc.lib(), batch=1, qh=32, kvh=8, pages=1000, page_stride=8 * 16 * 128,
                          workspace=ws, ws_bytes=size) != 0
            assert "workspace" in tmc.last_error()
    for bad in ((0, 8, 32, 8, 128, 1000), (1, 0, 32, 8, 128, 1000), (1, 8, 33, 8, 128, 1000),
                (1, 8, 32, 8, 128, 0), (1, 257, 32, 8, 128, 1000), (1, 8, 32, 0, 128, 1000)):
        assert tmc.tree_attention_workspace_bytes(*bad) == 0


def draw(lib, logits=P, dtype=1, stride=1000, uniforms=P, tokens=P, rows=4, vocab=1000, workspace=P,
         ws_bytes=HUGE):
    return lib.tmc_sample(logits, dtype, stride, None, None, None, None, uniforms, tokens, None, rows,
                          vocab, workspace, ws_bytes, None)


@pytest.mark.parametrize("change,text", [
    (dict(logits=None), "null"), (dict(uniforms=None), "null"), (dict(tokens=None), "null"),
    (dict(dtype=2), "f32 or f16"), (dict(dtype=3), "f32 or f16"), (dict(stride=999), "shape"),
    (dict(stride=1 << 36), "shape"), (dict(rows=0), "shape"), (dict(rows=1 << 24), "shape"),
    (dict(vocab=0), "shape"), (dict(vocab=(1 << 20) + 1, stride=1 << 21), "shape"),
    (dict(logits=C.c_void_p(4098)), "aligned"), (dict(logits=C.c_void_p(4097), dtype=0), "aligned")])
def test_sample_refuses(tmc, change, text):
    assert draw(tmc.lib(), **change) != 0
    assert text in tmc.last_error()


def test_sample_needs_its_workspace(tmc):
    need = tmc.sample_workspace_bytes(4, 128000)
    if need:
        for ws, size in ((P, need - 1), (None, need), (ODD, need)):
            assert draw(tmc.lib(), vocab=128000, stride=128000, workspace=ws, ws_bytes=size) != 0
            assert "workspace" in tmc.last_error()
    assert tmc.sample_workspace_bytes(0, 32000) == 0
    assert tmc.sample_workspace_bytes(4, 0) == 0
    assert tmc.sample_workspace_bytes(4, (1 << 20) + 1) == 0


def accept(lib, drafted=P, parents=P, chosen=P, cached=None, path=P, accepted=P, emitted=P,
           lengths=None, batch=2, nodes=8):
    return lib.tmc_tree_accept(drafted, parents, chosen, None, None, cached, path, accepted, emitted,
                               lengths, batch, nodes, None)


@pytest.mark.parametrize("change,text", [
    *[({n: None}, "null") for n in ("drafted", "parents", "chosen", "path", "accepted", "emitted")],
    (dict(lengths=P), "cached"), (dict(batch=0), "batch"), (dict(batch=65536), "batch"),
    (dict(nodes=0), "nodes"), (dict(nodes=257), "nodes")])
def test_accept_refuses(tmc, change, text):
    assert accept(tmc.lib(), **change) != 0
    assert text in tmc.last_error()


def keep(lib, keys=(P,), values=(P,), tables=P, cached=P, path=P, accepted=P, dtype=0, batch=2,
         nodes=8, heads=2, d=128, page=16, pages=4, pool=8, page_stride=2 * 16 * 128,
         head_stride=16 * 128):
    k = (C.c_void_p * len(keys))(*[x.value if x else None for x in keys])
    v = (C.c_void_p * len(values))(*[x.value if x else None for x in values])
    return lib.tmc_tree_keep(k, v, len(keys), tables, cached, path, accepted, dtype, batch, nodes,
                             heads, d, page, pages, pool, page_stride, head_stride, None)


@pytest.mark.parametrize("change,text", [
    *[({n: None}, "null") for n in ("tables", "cached", "path", "accepted")],
    (dict(keys=(None,)), "null pool"), (dict(values=(P, None), keys=(P, P)), "null pool"),
    (dict(keys=(), values=()), "pools"), (dict(dtype=3), "dtype"), (dict(batch=0), "batch"),
    (dict(nodes=257), "nodes"), (dict(heads=0), "heads"), (dict(d=0), "head_dim"),
    (dict(d=1025, head_stride=1 << 20, page_stride=1 << 22), "head_dim"), (dict(page=0), "geometry"),
    (dict(pages=1 << 28), "geometry"), (dict(pool=0), "geometry"), (dict(head_stride=8), "stride"),
    (dict(page_stride=16 * 128), "stride"), (dict(keys=(C.c_void_p(4097),)), "aligned")])
def test_keep_refuses(tmc, change, text):
    assert keep(tmc.lib(), **change) != 0
    assert text in tmc.last_error()
