"""Workspaces of tree attention and sampling: shapes that share their work need one, and a call
without it, or with less, is refused before any device work."""
import ctypes as C

import pytest

P = C.c_void_p(4096)  # a 16-byte aligned address that no refused call reads
ODD = C.c_void_p(4104)


@pytest.mark.parametrize("batch,nodes,qh,kvh,dim,pages", [
    (1, 8, 32, 8, 128, 1000), (16, 16, 32, 8, 128, 300), (2, 100, 8, 1, 64, 500), (1, 1, 1, 1, 64, 100)])
def test_attention(tmc, batch, nodes, qh, kvh, dim, pages):
    need = tmc.tree_attention_workspace_bytes(batch, nodes, qh, kvh, dim, 16 * pages)
    assert need > 0
    for space, size in ((P, need - 1), (P, 0), (None, need), (ODD, need)):
        assert tmc.lib().tmc_tree_attention(
            P, P, P, P, P, None, P, None, P, 0, batch, nodes, qh, kvh, dim, 16, pages, 8,
            kvh * 16 * dim, 16 * dim, space, size, None) != 0
        assert "workspace" in tmc.last_error()


def test_attention_without(tmc):
    """One block a request: short ones, and head dims of the plain kernel."""
    assert tmc.tree_attention_workspace_bytes(1, 8, 32, 8, 128, 64) == 0
    assert tmc.tree_attention_workspace_bytes(1, 8, 32, 8, 96, 16000) == 0


@pytest.mark.parametrize("rows,vocab", [(1, 32000), (4, 128000), (64, 128000), (511, 32000),
                                        (1, 1 << 20)])
def test_sampling(tmc, rows, vocab):
    need = tmc.sample_workspace_bytes(rows, vocab)
    assert need > 0
    for space, size in ((P, need - 1), (P, 0), (None, need), (ODD, need)):
        assert tmc.lib().tmc_sample(P, 1, vocab, None, None, None, None, P, P, None, rows, vocab,
                                    space, size, None) != 0
        assert "workspace" in tmc.last_error()


def test_sampling_without(tmc):
    """A block a row: many of them, or short ones."""
    assert tmc.sample_workspace_bytes(512, 128000) == 0
    assert tmc.sample_workspace_bytes(1, 2000) == 0
