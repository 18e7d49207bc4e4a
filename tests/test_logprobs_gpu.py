"""Log probabilities, entropy and top alternatives against 64 bits.

Tolerances: x - m is one fp32 rounding of a number of the row's spread,
2^-24 spread, and so is the argument of each exponential, whose own result is
good to 2^-22; log S is rounded once, 2^-24 of at most 14, and off by the
relative error of S: together 2^-20 + 2^-22 spread absolute.  The entropy adds
T / S, whose terms carry the same relative errors times |x - m|, which is below
90 where the term counts.
"""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "GPU tests need a GPU"
    return t


def run(tmc, torch, logits, tokens, top, workspace=None):
    rows, vocab = logits.shape
    out = dict(logprob=torch.full((rows,), 5.0, device="cuda"),
               entropy=torch.full((rows,), 5.0, device="cuda"),
               top_tokens=torch.full((rows, top), -9, dtype=torch.int32, device="cuda"),
               top_logprobs=torch.full((rows, top), 5.0, device="cuda"))
    if workspace is None:
        workspace = torch.zeros(max(1, tmc.logprobs_workspace_bytes(rows, vocab, top) // 4),
                                device="cuda")
    tmc.logprobs(logits, tokens, out["logprob"], out["entropy"], out["top_tokens"],
                 out["top_logprobs"], workspace)
    return out


def check(torch, logits, tokens, top, out):
    x = logits.double()
    logp = x - torch.logsumexp(x, -1, keepdim=True)
    p = torch.exp(logp)
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    finite = x.masked_fill(~torch.isfinite(x), 0.0)
    spread = (finite.amax(-1) - finite.amin(-1)).clamp(max=2000.0)
    tolerance = 2.0 ** -20 + 2.0 ** -22 * spread
    given = (tokens >= 0) & (tokens < x.shape[1])
    want = logp.gather(1, tokens.clamp(0, x.shape[1] - 1).long()[:, None])[:, 0]
    got = out["logprob"].double()
    assert (got[~given] == 5.0).all()
    near = ((got - want).abs() <= tolerance) | ((got == want) & torch.isinf(want))
    assert near[given].all()
    assert ((out["entropy"].double() - entropy).abs() <= tolerance * 90).all()
    which = torch.sort(x, stable=True, dim=-1, descending=True).indices[:, :top]
    assert torch.equal(out["top_tokens"].long(), which)
    want = logp.gather(1, which)
    got = out["top_logprobs"].double()
    assert (((got - want).abs() <= tolerance[:, None]) | ((got == want) & torch.isinf(want))).all()


SHAPES = [(1, 1, 1), (1, 2, 2), (3, 7, 7), (2, 63, 5), (2, 64, 64), (2, 65, 64), (5, 100, 20),
          (1, 32000, 5), (16, 32000, 20), (7, 32003, 1), (300, 2049, 3), (2, 8192, 64),
          (2, 8193, 64), (3, 160001, 20), (1, 1000000, 64), (64, 4097, 0), (2000, 515, 4),
          (2100, 1900, 20), (2048, 2048, 64), (2047, 1025, 5), (3, 1024, 64),
          (300, 60000, 20), (511, 25000, 3)]


@pytest.mark.parametrize("rows,vocab,top", SHAPES)
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_matches_64_bits(tmc, torch, rows, vocab, top, dtype):
    g = torch.Generator(device="cuda")
    g.manual_seed(rows + vocab)
    logits = (torch.randn(rows, vocab, generator=g, device="cuda") * 3).to(getattr(torch, dtype))
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    tokens[rows // 2] = vocab if rows > 1 else tokens[0]
    tokens[-1] = -1 if rows > 2 else tokens[-1]
    workspace = torch.zeros(max(1, tmc.logprobs_workspace_bytes(rows, vocab, top) // 4), device="cuda")
    out = run(tmc, torch, logits, tokens, top, workspace)
    check(torch, logits, tokens, top, out)
    again = run(tmc, torch, logits, tokens, top, workspace)
    for name in out:
        assert torch.equal(out[name], again[name]), name


@pytest.mark.parametrize("vocab", [65, 3000, 32000, 70001])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "few", "masked", "peak", "halves"])
def test_ties_orders_and_masks(tmc, torch, vocab, kind):
    """Rows that are hard to rank: all equal, sorted either way, a handful of
    distinct values, nearly all masked, one token with all the probability, and
    the best ones all in one stretch."""
    i = torch.arange(vocab, device="cuda", dtype=torch.float32)
    row = {"equal": torch.full((vocab,), -3.25, device="cuda"),
           "rising": i * (80.0 / vocab), "falling": -i * (80.0 / vocab), "few": (i * 7919) % 3,
           "masked": torch.where(i % 97 == 13, i * 1e-3, -math.inf),
           "peak": torch.where(i == vocab // 3, 200.0, i * 1e-4),
           "halves": torch.where((i >= vocab // 2) & (i < vocab // 2 + 60), 9.0 + i * 1e-3, 0.0)}[kind]
    logits = torch.stack([row, row.roll(1)])
    tokens = torch.tensor([vocab // 3, 0], dtype=torch.int32, device="cuda")
    for top in (1, 20, 64):
        check(torch, logits, tokens, top, run(tmc, torch, logits, tokens, top))


def test_best_tokens_all_in_the_last_parts(tmc, torch):
    """A long rising row: the parts at its end hold far more good candidates
    than the join ranks at once."""
    vocab = 1000003
    logits = (torch.arange(vocab, device="cuda") * (60.0 / vocab))[None]
    tokens = torch.tensor([vocab - 1], dtype=torch.int32, device="cuda")
    for top in (5, 64):
        check(torch, logits, tokens, top, run(tmc, torch, logits, tokens, top))


@pytest.mark.parametrize("rows,vocab", [(600, 32003), (3, 32003), (600, 5000)])
@pytest.mark.parametrize("top", [1, 20, 64])
@pytest.mark.parametrize("order", ["rising", "falling", "equal", "steps"])
def test_rows_that_fill_the_candidates(tmc, torch, rows, vocab, top, order):
    """Rows in whose every part all elements, none, or hundreds of equal ones reach
    the best so far."""
    at = torch.arange(vocab, device="cuda", dtype=torch.float32)
    row = {"rising": at / vocab, "falling": -at / vocab, "equal": torch.zeros_like(at) + 0.5,
           "steps": torch.floor(at / 300)}[order]
    logits = (row[None] + torch.arange(rows, device="cuda")[:, None] / 7).contiguous()
    tokens = torch.arange(rows, dtype=torch.int32, device="cuda") % vocab
    check(torch, logits, tokens, top, run(tmc, torch, logits, tokens, top))


def test_rows_without_a_distribution(tmc, torch):
    """NaN, +inf and empty rows: NaN log probabilities, the tokens still in the
    greedy order, and their neighbours untouched by it."""
    vocab, top = 5000, 4
    logits = torch.randn(6, vocab, device="cuda")
    logits[1, 77] = math.nan
    logits[2, 4000] = math.inf
    logits[3] = -math.inf
    logits[4] = math.nan
    tokens = torch.zeros(6, dtype=torch.int32, device="cuda")
    out = run(tmc, torch, logits, tokens, top)
    for r in (1, 2, 3, 4):
        assert math.isnan(out["logprob"][r]) and math.isnan(out["entropy"][r]), r
    good = torch.tensor([0, 5], device="cuda")
    check(torch, logits[good], tokens[good], top, {k: v[good] for k, v in out.items()})
    clean = logits[1].nan_to_num(-math.inf)
    assert out["top_tokens"][1].tolist() == torch.sort(clean, stable=True, descending=True).indices[:top].tolist()
    assert out["top_tokens"][2, 0] == 4000
    assert out["top_tokens"][3].tolist() == [0, 1, 2, 3]
    assert out["top_tokens"][4].tolist() == [-1] * 4
    assert out["top_logprobs"][4].tolist() == [-math.inf] * 4
    assert torch.isnan(out["top_logprobs"][1:4]).all()
    single = torch.full((1, 9), math.nan, device="cuda")
    single[0, 6], single[0, 2] = 1.0, -math.inf
    got = run(tmc, torch, single, tokens[:1], 4)
    assert got["top_tokens"].tolist() == [[6, 2, -1, -1]]
    assert got["top_logprobs"][0, 2:].tolist() == [-math.inf] * 2


def test_strided_rows_and_parts(tmc, torch):
    """Rows of a wider buffer at odd offsets; no tokens, no entropy, no
    alternatives; the greedy token is tmc_argmax_f32's."""
    wide = torch.randn(9, 40007, device="cuda")
    for low, vocab in ((0, 40007), (1, 32000), (3, 4099), (7, 1)):
        logits = wide[:, low:low + vocab]
        tokens = torch.full((9,), vocab - 1, dtype=torch.int32, device="cuda")
        top = min(5, vocab)
        out = run(tmc, torch, logits, tokens, top)
        check(torch, logits.contiguous(), tokens, top, out)
        greedy = torch.empty(9, dtype=torch.int32, device="cuda")
        tmc.argmax(logits.contiguous(), greedy)
        assert torch.equal(greedy, out["top_tokens"][:, 0])
        ws = torch.zeros(max(1, tmc.logprobs_workspace_bytes(9, vocab, top) // 4), device="cuda")
        entropy = torch.zeros(9, device="cuda")
        tmc.logprobs(logits, None, None, entropy, workspace=ws)
        assert torch.equal(entropy, out["entropy"])
        lone = torch.zeros(9, device="cuda")
        tmc.logprobs(logits, tokens, lone, workspace=ws)
        assert torch.equal(lone, out["logprob"])


def test_one_workspace_for_many_shapes(tmc, torch):
    shapes = [(16, 32000, 20), (1, 160000, 5), (300, 9000, 1), (2, 100, 64), (16, 32000, 20)]
    ws = torch.zeros(max(tmc.logprobs_workspace_bytes(*s) for s in shapes) // 4 + 1, device="cuda")
    for rows, vocab, top in shapes:
        logits = torch.randn(rows, vocab, device="cuda")
        tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        check(torch, logits, tokens, top, run(tmc, torch, logits, tokens, top, ws))


def test_graph_replays(tmc, torch):
    rows, vocab, top = 5, 32000, 7
    logits = torch.randn(rows, vocab, device="cuda")
    tokens = torch.arange(rows, dtype=torch.int32, device="cuda")
    ws, other = (torch.zeros(tmc.logprobs_workspace_bytes(rows, vocab, top) // 4 + 1, device="cuda")
                 for _ in range(2))
    lp, en = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    tt = torch.zeros(rows, top, dtype=torch.int32, device="cuda")
    tl = torch.zeros(rows, top, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tmc.logprobs(logits, tokens, lp, en, tt, tl, ws)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tmc.logprobs(logits, tokens, lp, en, tt, tl, ws)
    for step in range(5):
        logits.copy_(torch.randn(rows, vocab, device="cuda") * (1 + step))
        eager = run(tmc, torch, logits, tokens, top, other)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((lp, en, tt, tl), eager.values()):
            assert torch.equal(a, b), step


def test_wrappers_refuse(tmc, torch):
    logits, tokens = torch.zeros(2, 50, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    out = torch.zeros(2, device="cuda")
    tt, tl = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, 3, device="cuda")
    for args, text in (((logits.cpu(), tokens, out), "current GPU"), ((logits, tokens.cpu(), out), "current GPU"),
                       ((logits.t(), tokens, out), "adjacent"), ((logits, tokens.long(), out), "tokens must"),
                       ((logits, tokens[:1], out), "tokens holds"), ((logits, tokens, None), "go together"),
                       ((logits, tokens, out, None, tt, None), "top_logprobs"),
                       ((logits, tokens, out, None, tt, tl[:, :2].contiguous()), "rows, top"),
                       ((logits.bfloat16(), tokens, out), "f32 or f16"),
                       ((logits.double(), tokens, out), "f32 or f16")):
        with pytest.raises(RuntimeError, match=text):
            tmc.logprobs(*args)
