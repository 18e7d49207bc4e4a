"""Rows that a wave takes alone (short vocabularies): orders, ties and masks that fill
a wave's candidates, rows of one, two and three parts, and rows without a distribution.
Tolerances as in test_logprobs_gpu."""
import math

import pytest

from tests.test_logprobs_gpu import check, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "GPU tests need a GPU"
    return t


def rows_of(torch, kind, rows, vocab):
    i = torch.arange(vocab, device="cuda", dtype=torch.float32)
    r = torch.arange(rows, device="cuda", dtype=torch.float32)[:, None]
    return {"equal": (r * 0.0 + 0.5).expand(rows, vocab), "rising": i * (40.0 / vocab) + r * 0.0,
            "falling": -i * (40.0 / vocab) + r * 0.0, "few": (i * 7919 + r) % 3,
            "steps": torch.floor(i / 150) + r * 0.0, "zeros": torch.where((i + r) % 2 == 0, 0.0, -0.0),
            # of every row all but one in 97 masked, and all but 70 at its end
            "masked": torch.where((i + r) % 97 == 13, i * 1e-3, -math.inf),
            "tail": torch.where(i >= vocab - 70, i * 1e-2, -math.inf) + r * 0.0}[kind].contiguous()


@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "few", "steps", "zeros", "masked", "tail"])
@pytest.mark.parametrize("rows,vocab", [(3, 1000), (3, 1024), (700, 129), (2100, 1900), (2048, 2048),
                                        (2050, 1025)])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_short_rows(tmc, torch, kind, rows, vocab, dtype):
    logits = rows_of(torch, kind, rows, vocab).to(getattr(torch, dtype))
    tokens = torch.arange(rows, dtype=torch.int32, device="cuda") * 31 % vocab
    for top in (0, 1, 20, 64):
        check(torch, logits, tokens, top, run(tmc, torch, logits, tokens, top))


@pytest.mark.parametrize("rows,vocab", [(6, 1000), (2048, 2000)])
def test_short_rows_without_a_distribution(tmc, torch, rows, vocab):
    top = 5
    g = torch.Generator(device="cuda")
    g.manual_seed(rows)
    logits = torch.randn(rows, vocab, generator=g, device="cuda")
    logits[1, vocab - 1] = math.nan
    logits[2, vocab // 2] = math.inf
    logits[3] = -math.inf
    logits[4] = math.nan
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    out = run(tmc, torch, logits, tokens, top)
    for r in (1, 2, 3, 4):
        assert math.isnan(out["logprob"][r]) and math.isnan(out["entropy"][r]), r
    good = torch.tensor([0, 5, rows - 1], device="cuda")
    check(torch, logits[good], tokens[good], top, {k: v[good] for k, v in out.items()})
    clean = logits[1].nan_to_num(-math.inf)
    assert out["top_tokens"][1].tolist() == torch.sort(clean, stable=True, descending=True).indices[:top].tolist()
    assert out["top_tokens"][2, 0] == vocab // 2
    assert out["top_tokens"][3].tolist() == list(range(top))
    assert out["top_tokens"][4].tolist() == [-1] * top
    assert out["top_logprobs"][4].tolist() == [-math.inf] * top
