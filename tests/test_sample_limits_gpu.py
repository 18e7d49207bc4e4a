"""Sampling at the most tokens that it takes, 2^20: every part sum of a row is in use, and the
digits' weights have the fewest bits."""
import pytest
import torch

from test_sample_cuts_gpu import check_draws, noise

pytestmark = pytest.mark.gpu

MOST = 1 << 20


@pytest.mark.parametrize("rows", [512, 3])
@pytest.mark.parametrize("vocab", [MOST, MOST - 1, MOST - 2047])
def test_most_tokens(tmc, rows, vocab):
    row = noise(vocab, 41, 3.0, 0.5, torch.float16)
    row[-3:] = torch.tensor([9.0, -40.0, 12.0])
    for settings in (dict(), dict(top_p=0.97), dict(top_k=400), dict(top_p=0.9, min_p=1e-3),
                     dict(temperature=0.4, top_k=1024, top_p=0.99)):
        check_draws(tmc, row, rows, 42, **settings)


@pytest.mark.parametrize("rows", [512, 3])
@pytest.mark.parametrize("settings", [dict(), dict(top_p=0.61), dict(top_k=300000),
                                      dict(top_k=5000, top_p=0.7, min_p=0.9)])
def test_most_tokens_all_alike(tmc, rows, settings):
    row = torch.full((MOST,), -2.5, dtype=torch.float16)
    check_draws(tmc, row, rows, 43, **settings)
    row[::2] = -2.75
    check_draws(tmc, row, rows, 44, **settings)
