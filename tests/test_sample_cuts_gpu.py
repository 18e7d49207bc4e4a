"""Sampling where a cut is hard to find: long runs of equal logits, logits that are great
next to the temperature.  Rows hold the same logits and settings and differ in their random
numbers, so that draws reach all that stays."""
import numpy as np
import pytest
import torch

from sample_helpers import kept_weights, single

pytestmark = pytest.mark.gpu


def check_draws(tmc, row, rows, seed, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Tokens, either of two neighbours where a number lies on their border: n running sums of 64
    bits are off by n 2^-53 of the whole, the kernel's weights by 2^-44 of the greatest each,
    which is 2^-44 n / n' of the whole for n' of at least half the greatest, here 2^-42 at most
    (2^20 tokens of alike weights have borders on multiples of 2^-20, as the numbers).
    Probabilities as in test_sample_gpu.check()."""
    weight = kept_weights(row.float().numpy(), temperature, top_k, top_p, min_p)
    sums = np.cumsum(weight)
    u = np.random.default_rng(seed).random(rows).astype(np.float32)
    u[0] = 0.0
    u[-1] = np.float32(1.0 - 2.0 ** -24)
    want = np.searchsorted(sums, u.astype(np.float64) * sums[-1], side="right")
    logits = row.cuda().expand(rows, -1).contiguous()
    full = lambda v, t: torch.full((rows,), v, dtype=t, device="cuda")  # noqa: E731
    tokens, shares = full(-7, torch.int32), full(-7.0, torch.float32)
    space = torch.zeros(tmc.sample_workspace_bytes(rows, len(row)) // 4 + 4, device="cuda")
    tmc.sample(logits, torch.from_numpy(u).cuda(), tokens, full(temperature, torch.float32),
               full(top_k, torch.int32), full(top_p, torch.float32), full(min_p, torch.float32),
               probability=shares, workspace=space)
    got = tokens.cpu().numpy()
    assert ((got >= 0) & (got < len(row))).all()
    kept = np.cumsum(weight > 0)
    low, high = np.minimum(got, want), np.maximum(got, want)
    on_border = (np.abs(u * sums[-1] - sums[low]) <= (len(row) * 2.0 ** -53 + 2.0 ** -42) * sums[-1]) \
        & (kept[high] - kept[low] == 1) & (weight[got] > 0)
    bad = (got != want) & ~on_border
    assert not bad.any(), f"{bad.sum()} of {rows} differ, {(weight[got] == 0).sum()} are cut off"
    share = weight[got] / sums[-1]
    off = np.abs(shares.cpu().numpy() - share)
    assert (off <= 2.0 ** -23 * share + 2.0 ** -34).all()
    assert single(share[0]) > 0


def noise(vocab, seed, spread, offset, dtype):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(vocab, generator=gen) * spread + offset).to(dtype)


# (rows of one block each, and of several)
ROWS = [512, 40]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("vocab,spread,offset,dtype,top_p", [
    (128000, 0.1, 10.0, torch.float16, 0.5),
    (128000, 0.05, 5.0, torch.float16, 0.5),
    (128000, 0.1, -300.0, torch.float16, 0.7),
    (40000, 0.01, 1000.0, torch.float32, 0.9),
    (40000, 0.3, 1e6, torch.float32, 0.5),
    (40000, 0.3, -2e6, torch.float32, 0.8),
    (40000, 0.0, 7.0, torch.float32, 0.3),
])
def test_alike_far_from_zero(tmc, rows, vocab, spread, offset, dtype, top_p):
    """Thousands of equal logits at the cut, whose bins' numbers grow with the offset."""
    row = noise(vocab, 21, spread, offset, dtype)
    check_draws(tmc, row, rows, 22, top_p=top_p)
    check_draws(tmc, row, rows, 23, top_k=700, top_p=top_p)
    check_draws(tmc, row, rows, 24, temperature=0.25, top_p=top_p)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("top_p", [0.1, 0.5, 0.9, 0.999])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_few_great_values(tmc, rows, top_p, dtype):
    gen = torch.Generator().manual_seed(25)
    row = torch.randint(3, 8, (30011,), generator=gen).to(dtype)
    check_draws(tmc, row, rows, 26, top_p=top_p)
    check_draws(tmc, row, rows, 27, temperature=3.0, top_p=top_p)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("settings", [dict(top_p=0.9), dict(top_k=50, top_p=0.9), dict(top_k=900),
                                      dict(min_p=0.01), dict()])
def test_forbidden_blocks(tmc, rows, settings):
    """A third of the vocabulary forbidden by a great negative number, whole blocks of it."""
    for least in (-1e4, -1e9, -1e30, torch.finfo(torch.float32).min):
        row = noise(30011, 28, 2.0, 0.0, torch.float32)
        row[4000:14000] = least
        check_draws(tmc, row, rows, 29, **settings)
        check_draws(tmc, row, rows, 30, temperature=0.1, **settings)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("vocab,spread,offset,dtype", [
    (46060, 1.2, 1203.0, torch.float16),     # steps of 1 between logits
    (46060, 12.0, -1e4, torch.float16),
    (112000, 0.008, -37300.0, torch.float32),
    (112000, 0.008, 5e4, torch.float32),
    (30011, 0.5, 3e5, torch.float32),
])
@pytest.mark.parametrize("top_k", [300, 1000, 1024])
def test_top_k_among_equals_far_from_zero(tmc, rows, vocab, spread, offset, dtype, top_k):
    """The cut by number inside a run of more equals than a list holds, at logits whose
    neighbouring floats lie many finer bins apart."""
    row = noise(vocab, 31, spread, offset, dtype)
    check_draws(tmc, row, rows, 32, top_k=top_k)
    check_draws(tmc, row, rows, 33, top_k=top_k, top_p=0.6)
    check_draws(tmc, row, rows, 34, temperature=0.5, top_k=top_k, min_p=1e-4)


PLATEAUS = [(1, 0.0), (20000, -0.64523), (617, -0.90103), (40000, -1.37627)]


def plateaus(shuffled):
    row = torch.cat([torch.full((n,), v) for n, v in PLATEAUS])
    return row[torch.randperm(len(row), generator=torch.Generator().manual_seed(35))] if shuffled else row


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("edge", [1, 2, 3])
@pytest.mark.parametrize("min_p", [0.0, 0.01, 0.3, 0.45, 0.52])
def test_cuts_next_to_gaps(tmc, rows, edge, min_p):
    """top_p just before and behind the end of a run of equals with nothing for many bins
    behind it, alone and where min_p is far behind, in the gaps or before the cut."""
    row = plateaus(shuffled=edge == 3)
    weight = np.exp(np.array([single(v) for _, v in PLATEAUS])) * [n for n, _ in PLATEAUS]
    at = weight[:edge].sum() / weight.sum()
    for off in np.geomspace(2e-6, 6e-4, 24):
        for top_p in (at - off, at + off):
            if 0 < top_p < 1:
                check_draws(tmc, row, rows, 36, top_p=top_p, min_p=min_p)


@pytest.mark.parametrize("rows", ROWS)
def test_top_p_with_min_p_next_to_a_gap(tmc, rows):
    """Three tokens behind the cut stayed, and 14000 was drawn for 13998 with 0.7."""
    row = plateaus(shuffled=False)
    check_draws(tmc, row, rows, 37, top_p=0.50328, min_p=0.01)
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    full = lambda v: torch.full((rows,), v, device="cuda")  # noqa: E731
    space = torch.zeros(tmc.sample_workspace_bytes(rows, len(row)) // 4 + 4, device="cuda")
    tmc.sample(row.cuda().expand(rows, -1).contiguous(), full(0.7), tokens, top_p=full(0.50328),
               min_p=full(0.01), workspace=space)
    assert (tokens == 13998).all()


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("min_p", [0.5, 1.0, 3.0])
@pytest.mark.parametrize("vocab", [50, 9001])
def test_infinite_temperature_with_min_p(tmc, rows, min_p, vocab):
    """All weights are 1, and min-p keeps them all."""
    row = noise(vocab, 38, 2.0, 1.0, torch.float32)
    row[::3] = float("-inf")
    for more in (dict(), dict(top_k=7), dict(top_p=0.613), dict(top_k=1500, top_p=0.8)):
        check_draws(tmc, row, rows, 39, temperature=float("inf"), min_p=min_p, **more)
