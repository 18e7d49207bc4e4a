"""Sampling from given random numbers, against 64 bits."""
import math

import numpy as np
import pytest
import torch

from sample_helpers import draw

pytestmark = pytest.mark.gpu

NEUTRAL = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
STYLES = {
    "temperature": [dict(temperature=t) for t in (0.3, 0.7, 1.0, 2.5)],
    "top_k": [dict(temperature=0.8, top_k=k) for k in (1, 2, 40, 1000)],
    "top_p": [dict(top_p=p) for p in (0.05, 0.5, 0.9, 0.99)],
    "min_p": [dict(min_p=p) for p in (0.001, 0.05, 0.5, 1.0)],
    "all": [dict(temperature=t, top_k=k, top_p=p, min_p=m) for t, k, p, m in (
        (0.7, 50, 0.9, 0.02), (1.3, 500, 0.95, 0.001), (1.0, 3, 0.5, 0.3), (0.2, 100000, 0.8, 0.0))],
    "greedy": [dict(temperature=t) for t in (0.0, -1.0, 1e-6, math.nan)],
    "odd": [dict(top_p=0.0), dict(min_p=7.0), dict(temperature=math.inf, top_k=5),
            dict(top_p=math.nan, min_p=math.nan, top_k=-3)],
    "mixed": [dict(), dict(temperature=0.0), dict(top_k=20), dict(top_p=0.9), dict(min_p=0.1),
              dict(temperature=0.5, top_k=64, top_p=0.95, min_p=0.01)],
}


def run(tmc, logits, u, settings, probability=True, stream=None, workspace=None, tokens=None):
    rows, vocab = logits.shape
    column = lambda name, dtype: torch.tensor(  # noqa: E731
        [{**NEUTRAL, **s}[name] for s in settings], dtype=dtype, device="cuda")
    if tokens is None:
        tokens = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    shares = torch.full((rows,), -7.0, device="cuda") if probability else None
    if workspace is None:
        workspace = torch.zeros(max(4, tmc.sample_workspace_bytes(rows, vocab) // 4 + 1),
                                device="cuda")
    args = {n: column(n, d) for n, d in (("temperature", torch.float32), ("top_k", torch.int32),
                                         ("top_p", torch.float32), ("min_p", torch.float32))}
    tmc.sample(logits, torch.as_tensor(u, dtype=torch.float32).cuda(), tokens, **args,
               probability=shares, workspace=workspace, stream=stream)
    return tokens, shares


def check(tmc, logits, u, settings, **more):
    """Tokens exactly; a probability is a quotient in 64 bits rounded to 32 (2^-24),
    its weights multiples of 2^-34 or less of the greatest, its sum at least 1."""
    tokens, shares = run(tmc, logits, u, settings, **more)
    x = logits.float().cpu().numpy()
    for r, s in enumerate(settings):
        token, share = draw(x[r], float(u[r]), **{**NEUTRAL, **s})
        assert int(tokens[r]) == token, f"row {r} {s} u {float(u[r])}"
        got = float(shares[r])
        assert (math.isnan(got) and math.isnan(share)) or \
            abs(got - share) <= 2.0 ** -23 * share + 2.0 ** -34, f"row {r} {s}"


def numbers(rows, seed):
    u = np.random.default_rng(seed).random(rows).astype(np.float32)
    u[0] = 0.0
    if rows > 1:
        u[1] = np.float32(1.0 - 2.0 ** -24)
    return u


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 1000, 4097, 32000, 50257, 131075])
@pytest.mark.parametrize("style", list(STYLES))
def test_sample(tmc, vocab, style):
    kinds = STYLES[style]
    rows = 2 * len(kinds)
    gen = torch.Generator().manual_seed(vocab)
    logits = torch.randn(rows, vocab, generator=gen) * 3.0
    check(tmc, logits.cuda(), numbers(rows, vocab), kinds + kinds)


@pytest.mark.parametrize("rows,vocab", [(1, 32000), (7, 32000), (64, 8000), (300, 1000), (600, 2000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_rows(tmc, rows, vocab, dtype):
    gen = torch.Generator().manual_seed(rows)
    logits = (torch.randn(rows, vocab, generator=gen) * 3.0).to(dtype)
    kinds = sum(STYLES.values(), [])
    check(tmc, logits.cuda(), numbers(rows, rows), [kinds[r % len(kinds)] for r in range(rows)])


@pytest.mark.parametrize("style", ["temperature", "top_k", "top_p", "min_p", "all", "mixed"])
@pytest.mark.parametrize("spread", [0.0, 1e-3, 0.3, 30.0, 1e4])
def test_flat_and_steep_rows(tmc, style, spread):
    """Rows that are nearly or all alike, whose cuts fall among very many tokens, and
    rows of a few tokens."""
    kinds = STYLES[style]
    gen = torch.Generator().manual_seed(5)
    logits = torch.randn(len(kinds), 20011, generator=gen) * spread
    check(tmc, logits.cuda(), numbers(len(kinds), 3), kinds)


@pytest.mark.parametrize("rows,vocab", [(520, 9001), (3, 131072)])
@pytest.mark.parametrize("spread", [3e-6, 1e-3, 0.05, 0.5])
def test_cuts_among_many(tmc, rows, vocab, spread):
    """More tokens near the cut than a list holds, in rows of one block and of several."""
    kinds = [dict(top_p=0.9), dict(top_k=900, top_p=0.7), dict(top_p=0.3, min_p=0.2),
             dict(top_k=1000), dict(top_p=0.999), dict(top_k=1500, top_p=0.5)]
    gen = torch.Generator().manual_seed(11)
    logits = torch.randn(rows, vocab, generator=gen) * spread - 1.0
    check(tmc, logits.cuda(), numbers(rows, 12), [kinds[r % len(kinds)] for r in range(rows)])


@pytest.mark.parametrize("style", ["temperature", "top_k", "top_p", "min_p", "all", "greedy"])
def test_equal_logits(tmc, style):
    """Few different values: every cut falls inside a run of equals."""
    kinds = STYLES[style] * 3
    gen = torch.Generator().manual_seed(6)
    logits = torch.randint(-2, 3, (len(kinds), 30011), generator=gen).float()
    logits[1::2] = logits[1::2].half().float() * 0.5
    check(tmc, logits.cuda(), numbers(len(kinds), 4), kinds)
    check(tmc, logits.half().cuda(), numbers(len(kinds), 4), kinds)


@pytest.mark.parametrize("style", list(STYLES))
@pytest.mark.parametrize("vocab", [7, 5000, 40000])
def test_forbidden_and_special(tmc, style, vocab):
    kinds = STYLES[style] * 3
    rows = len(kinds)
    gen = torch.Generator().manual_seed(7)
    logits = torch.randn(rows, vocab, generator=gen) * 2.0
    logits[:, ::3] = -math.inf
    logits[1, 1::2] = math.nan
    logits[2, vocab // 2] = math.inf
    logits[2, 1] = math.inf
    logits[3] = -math.inf
    if rows > 4:
        logits[4] = math.nan
        logits[5, 1:] = -math.inf
        logits[6] = torch.finfo(torch.float32).min
        logits[7, 1::2] = torch.finfo(torch.float32).min
        logits[8] = torch.finfo(torch.float32).max
        logits[9, 0], logits[9, 1] = -0.0, 0.0
        logits[10] = -math.inf
        logits[10, 5] = math.nan
        logits[10, 6] = -4.0
    check(tmc, logits.cuda(), numbers(rows, 8), kinds)


@pytest.mark.parametrize("u", [-1.0, math.nan, 1.0, 2.0, math.inf])
def test_numbers_out_of_range(tmc, u):
    logits = torch.randn(3, 999, generator=torch.Generator().manual_seed(1)).cuda()
    kinds = [dict(), dict(top_k=7), dict(top_p=0.6)]
    tokens, _ = run(tmc, logits, [u] * 3, kinds)
    x = logits.cpu().numpy()
    for r, s in enumerate(kinds):
        assert int(tokens[r]) == draw(x[r], u, **{**NEUTRAL, **s})[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("gap", [1, 3, 64])
def test_strided_rows(tmc, dtype, gap):
    kinds = STYLES["mixed"]
    gen = torch.Generator().manual_seed(9)
    wide = (torch.randn(len(kinds), 5003 + gap + 1, generator=gen) * 3.0).to(dtype)
    wide[:, 5004:] = 1000.0  # what lies between the rows is nobody's
    wide[:, 0] = 1000.0
    check(tmc, wide.cuda()[:, 1:5004], numbers(len(kinds), 10), kinds)


def test_every_token_gets_its_share(tmc):
    """Numbers over the whole of [0, 1) reach every token in order, each its share."""
    rows, weights = 4096, torch.tensor([1.0, 4.0, 0.0, 2.0, 8.0, 1.0])
    u = (torch.arange(rows) + 0.5) / rows
    tokens, shares = run(tmc, weights.log().expand(rows, -1).contiguous().cuda(), u, [dict()] * rows)
    tokens = tokens.cpu()
    assert (tokens[1:] >= tokens[:-1]).all()
    counts = torch.bincount(tokens.long(), minlength=6).double()
    # log and exp of 32 bits: shares off by 2^-22 at most, a border by less than a number
    assert ((counts - rows * weights.double() / 16).abs() <= 1).all()


def test_neutral_settings(tmc):
    """No arrays are neutral arrays."""
    logits = torch.randn(5, 3001, generator=torch.Generator().manual_seed(2)).cuda()
    u = torch.rand(5, generator=torch.Generator().manual_seed(3)).cuda()
    tokens = torch.zeros(5, dtype=torch.int32, device="cuda")
    space = torch.zeros(max(4, tmc.sample_workspace_bytes(5, 3001)), dtype=torch.uint8, device="cuda")
    tmc.sample(logits, u, tokens, workspace=space)
    assert torch.equal(tokens, run(tmc, logits, u, [dict()] * 5, probability=False)[0])


def test_same_bits_every_time(tmc):
    kinds = STYLES["mixed"] * 4
    logits = (torch.randn(len(kinds), 32000, generator=torch.Generator().manual_seed(4)) * 2).cuda()
    u = numbers(len(kinds), 5)
    first = run(tmc, logits, u, kinds)
    for _ in range(5):
        again = run(tmc, logits, u, kinds)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_one_workspace_for_all(tmc):
    shapes = [(1, 100000), (16, 32000), (3, 50), (200, 9000)]
    space = torch.zeros(max(tmc.sample_workspace_bytes(*s) for s in shapes) // 4 + 4, device="cuda")
    kinds = STYLES["all"]
    for turn in range(2):
        for rows, vocab in shapes:
            logits = torch.randn(rows, vocab, generator=torch.Generator().manual_seed(vocab)) * 3
            check(tmc, logits.cuda(), numbers(rows, turn), [kinds[r % 4] for r in range(rows)],
                  workspace=space)


def test_captured_and_on_a_stream(tmc):
    rows, vocab = 6, 32000
    kinds = STYLES["mixed"]
    logits = (torch.randn(rows, vocab, generator=torch.Generator().manual_seed(4)) * 2).cuda()
    u = torch.from_numpy(numbers(rows, 5)).cuda()
    space = torch.zeros(tmc.sample_workspace_bytes(rows, vocab) // 4 + 4, device="cuda")
    f32 = lambda n: torch.tensor([{**NEUTRAL, **s}[n] for s in kinds], device="cuda")  # noqa: E731
    heat, share, least = (f32(n).float() for n in ("temperature", "top_p", "min_p"))
    k = f32("top_k").int()
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    want, _ = run(tmc, logits, u, kinds)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tmc.sample(logits, u, tokens, temperature=heat, top_k=k, top_p=share, min_p=least,
                   workspace=space)
    for _ in range(3):
        tokens.fill_(-5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tokens, want)
    side = torch.cuda.Stream()
    tokens.fill_(-5)
    side.wait_stream(torch.cuda.current_stream())
    tmc.sample(logits, u, tokens, temperature=heat, top_k=k, top_p=share, min_p=least,
               workspace=space, stream=side)
    side.synchronize()
    assert torch.equal(tokens, want)


def test_refusals(tmc):
    logits, u = torch.zeros(2, 100, device="cuda"), torch.zeros(2, device="cuda")
    tokens = torch.full((2,), -7, dtype=torch.int32, device="cuda")
    for bad in (dict(logits=logits.double()), dict(logits=logits.t()), dict(logits=logits[0]),
                dict(logits=logits.cpu()), dict(u=u.cpu()), dict(u=u[:1]), dict(tokens=tokens.long()),
                dict(top_k=u), dict(temperature=u.half()), dict(min_p=u[:1]), dict(top_p=u.double())):
        args = dict(logits=logits, u=u, tokens=tokens, **{k: v for k, v in bad.items()
                                                          if k not in ("logits", "u", "tokens")})
        args.update({k: v for k, v in bad.items() if k in ("logits", "u", "tokens")})
        with pytest.raises(tmc.TmcError):
            tmc.sample(args.pop("logits"), args.pop("u"), args.pop("tokens"), **args)
    assert (tokens == -7).all()


def test_two_at_once(tmc):
    """On two streams with a workspace each, neither waiting for the other."""
    rows, vocab, kinds = 9, 50000, STYLES["all"]
    settings = [kinds[r % len(kinds)] for r in range(rows)]
    logits = [torch.randn(rows, vocab, generator=torch.Generator().manual_seed(30 + i)) * 3
              for i in range(2)]
    u = [numbers(rows, 40 + i) for i in range(2)]
    want = [run(tmc, x.cuda(), n, settings) for x, n in zip(logits, u)]
    f32 = lambda n: torch.tensor([{**NEUTRAL, **s}[n] for s in settings], device="cuda")  # noqa: E731
    heat, share, least = (f32(n).float() for n in ("temperature", "top_p", "min_p"))
    k = f32("top_k").int()
    sides = [dict(x=x.cuda(), u=torch.from_numpy(n).cuda(), stream=torch.cuda.Stream(),
                  tokens=torch.full((rows,), -5, dtype=torch.int32, device="cuda"),
                  space=torch.zeros(tmc.sample_workspace_bytes(rows, vocab) // 4 + 4, device="cuda"))
             for x, n in zip(logits, u)]
    torch.cuda.synchronize()
    for _ in range(6):
        for s in sides:
            tmc.sample(s["x"], s["u"], s["tokens"], temperature=heat, top_k=k, top_p=share,
                       min_p=least, workspace=s["space"], stream=s["stream"])
    torch.cuda.synchronize()
    for s, (tokens, _) in zip(sides, want):
        assert torch.equal(s["tokens"], tokens)
