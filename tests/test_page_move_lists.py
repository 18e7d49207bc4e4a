"""Lists of page moves in other containers than lists: read on the host, wherever
they lie, and checked at their full width."""
import numpy as np
import pytest
import torch

MOVES = [(0, 1, 2, 16), (1, 1, 3, 4), (1, 2, 1 << 3, 5)]  # the last page does not exist


@pytest.mark.parametrize("make", [
    lambda m: m, lambda m: torch.tensor(m), lambda m: torch.tensor(m, dtype=torch.int32),
    lambda m: np.array(m), lambda m: np.array(m, dtype=np.int32), tuple])
def test_containers_are_checked(tmc, make):
    with pytest.raises(RuntimeError, match="move 2 names a pool or page that does not exist"):
        tmc.page_moves(make(MOVES), 2, 8, 16)


@pytest.mark.parametrize("make", [torch.tensor, np.array])
def test_wide_numbers_are_not_cut(tmc, make):
    """2^32 + 1 cut to 32 bits would name page 1."""
    with pytest.raises(RuntimeError, match="overflow"):
        tmc.page_moves(make([(0, 2 ** 32 + 1, 2, 16)]), 1, 8, 16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_moves_on_the_device(tmc, dtype):
    moves = torch.tensor(MOVES, dtype=dtype, device="cuda")
    with pytest.raises(RuntimeError, match="does not exist"):
        tmc.page_moves(moves, 2, 8, 16)
    got = tmc.page_moves(moves[:2], 2, 8, 16)
    assert got.is_cuda and got.dtype is torch.int32 and torch.equal(got, moves[:2].int())


def test_more_moves_than_a_launch_takes_are_refused(tmc):
    """A block of 256 threads a move: 2^24 moves are 2^32 threads, which no launch takes."""
    import ctypes as C
    pool = (C.c_void_p * 1)(4096)
    for count in (1 << 24, (1 << 31) - 1):
        assert tmc.lib().tmc_move_pages(pool, pool, 1, C.c_void_p(4096), count, 0, 8, 2, 16, 128,
                                        2 * 16 * 128, 16 * 128, None) != 0
        assert "shape" in tmc.last_error()
