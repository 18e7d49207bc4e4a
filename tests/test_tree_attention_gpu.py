"""Attention of trees of drafted tokens over a paged cache, against 64 bits."""
import random

import numpy as np
import pytest
import torch

from tree_helpers import Forest

pytestmark = pytest.mark.gpu

SHAPES = [
    # cached, nodes, q heads, kv heads, dim, page
    ([0], 1, 4, 4, 128, 16),
    ([0, 1, 5], 3, 4, 2, 64, 4),
    ([300], 8, 32, 8, 128, 16),
    ([17, 64, 1000], 13, 8, 2, 64, 12),
    ([31, 32, 33, 63, 64, 65, 0], 33, 6, 2, 128, 16),
    ([100], 256, 8, 1, 64, 16),
    ([70], 65, 4, 4, 128, 1),
    ([15, 200], 40, 24, 2, 128, 7),
    ([5000, 129, 20000], 16, 8, 2, 128, 16),
    ([9000], 60, 8, 2, 64, 32),
    ([40, 3], 9, 71, 1, 128, 16),
    ([100, 7], 5, 4, 2, 96, 16),
    ([50, 0], 20, 2, 1, 256, 8),
    ([20], 4, 3, 1, 8, 5),
]


@pytest.mark.parametrize("cached,nodes,qh,kvh,dim,page", SHAPES)
def test_attention(tmc, cached, nodes, qh, kvh, dim, page):
    f = Forest(1, cached, nodes, qh, kvh, dim, page)
    t = f.device()
    f.attend(tmc, t)
    f.check(t)


@pytest.mark.parametrize("dim", [64, 128, 96])
def test_ragged_padded_and_strided(tmc, dim):
    cached = [12, 0, 700, 45, 333, 64]
    f = Forest(2, cached, 21, 8, 2, dim, 16, counts=[21, 1, 7, 0, 20, 5], active=5, gap=(24, 40))
    t = f.device()
    f.attend(tmc, t)
    f.check(t)


@pytest.mark.parametrize("dim", [64, 128, 96])
def test_no_counts_and_no_active(tmc, dim):
    f = Forest(3, [5, 90], 6, 4, 1, dim, 16)
    t = f.device()
    f.attend(tmc, t, counts=False, active=False)
    f.check(t)


@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("cached", [0, 1, 40, 1500])
def test_any_masks(tmc, dim, cached):
    """Bits that no tree has: nodes that see nothing, later nodes, bits behind the count."""
    rng = random.Random(4)
    nodes = 45
    sees = [[set() if i % 5 == 0 else {j for j in range(nodes) if rng.random() < 0.3}
             for i in range(nodes)]]
    f = Forest(4, [cached], nodes, 4, 2, dim, 16, counts=[41], sees=sees)
    t = f.device()
    f.attend(tmc, t)
    f.check(t)


@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_what_is_not_seen_changes_nothing(tmc, dim, value):
    f = Forest(5, [30, 500], 20, 8, 2, dim, 16)
    for r, c in enumerate(f.cached):
        for j in (3, 11, 19):
            f.k[r][c + j, :, 1] = np.nan
            f.v[r][c + j, :, ::3] = value
    # nodes that see one of them: NaN scores, so only the others are looked at
    t = f.device()
    f.attend(tmc, t)
    f.check(t)


@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_what_is_seen_shows(tmc, dim, value):
    f = Forest(6, [30, 500], 20, 8, 2, dim, 16)
    for r, c in enumerate(f.cached):
        f.v[r][c + 3, :, 5] = value
        f.v[r][7, 0, 9] = value
    t = f.device()
    f.attend(tmc, t)
    f.check(t)


@pytest.mark.parametrize("dim", [64, 128, 96])
def test_great_scores(tmc, dim):
    """Scores of up to a few thousand: one position takes all the weight."""
    f = Forest(7, [100, 900], 18, 8, 2, dim, 16)
    f.q *= np.float16(40.0)
    for x in f.k:
        x *= np.float16(8.0)
    t = f.device()
    f.attend(tmc, t)
    got = t["out"].float().cpu().numpy().reshape(f.batch, f.nodes, f.q_heads, f.dim)
    for r in range(f.batch):
        want, size = f.exact(r)
        # a score of 2^12 is off by 2^-10 in fp32 sums of D products, its weight by as much
        bound = 2.0 ** -10 * np.abs(want) + (2.0 ** -11 + 2.0 ** -8) * size + 2.0 ** -24
        assert (np.abs(got[r] - want) <= bound).all()


@pytest.mark.parametrize("dim", [64, 128, 96])
def test_requests_left_alone(tmc, dim):
    cached = [20, 33, 70, 5, 16]
    f = Forest(8, cached, 6, 4, 2, dim, 16)
    t = f.device()
    t["tables"][0, 1] = -1           # a page of the tree
    t["tables"][2, 0] = f.pages      # no such page
    t["cached"][3] = -1              # no such length
    t["cached"][4] = f.page * f.max_pages - 5  # one node too many for the capacity
    f.attend(tmc, t)
    for r in (0, 2, 3, 4):
        assert (t["out"][r] == 7.0).all(), r
    whole = t["out"][1].float().cpu().numpy().reshape(6, 4, dim)
    want, size = f.exact(1)
    bound = 2.0 ** -10 * np.abs(want) + (2.0 ** -11 + 2.0 ** -14) * size + 2.0 ** -24
    assert (np.abs(whole - want) <= bound).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_one_workspace_for_all(tmc, dim):
    """Launches of unlike shapes through one workspace, twice each: the same bits."""
    forests = [Forest(9 + i, *s) for i, s in enumerate([
        ([4000], 8, 8, 2, dim, 16), ([300, 2000, 17], 30, 8, 8, dim, 16),
        ([9000, 50], 3, 8, 1, dim, 16)])]
    space = max((f.workspace(tmc) for f in forests), key=lambda w: w.numel())
    first = []
    for turn in range(2):
        for i, f in enumerate(forests):
            t = f.device()
            f.attend(tmc, t, workspace=space)
            if turn == 0:
                f.check(t)
                first.append(t["out"].clone())
            else:
                assert torch.equal(first[i], t["out"])


@pytest.mark.parametrize("dim", [64, 128])
def test_captured(tmc, dim):
    f = Forest(12, [2500, 40], 12, 8, 2, dim, 16)
    t = f.device()
    space = f.attend(tmc, t)
    torch.cuda.synchronize()
    want = t["out"].clone()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            f.attend(tmc, t, workspace=space)
    torch.cuda.synchronize()
    for _ in range(3):
        t["out"].fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(t["out"], want)
        t["q"] += 0  # the program's own work between the replays


def test_on_a_stream(tmc):
    f = Forest(13, [800], 10, 8, 2, 128, 16)
    t = f.device()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    f.attend(tmc, t, workspace=f.workspace(tmc), stream=side)
    side.synchronize()
    f.check(t)


def test_refusals(tmc):
    f = Forest(14, [40], 4, 4, 2, 128, 16)
    t = f.device()
    for name, bad in (("q", t["q"].float()), ("masks", t["masks"].long()), ("cached", t["cached"].cpu()),
                      ("tables", t["tables"][:, ::2]), ("out", t["out"][:, :2])):
        with pytest.raises(tmc.TmcError):
            f.attend(tmc, dict(t, **{name: bad}))
    with pytest.raises(tmc.TmcError):
        f.attend(tmc, t, pool_pages=f.pages + 1)
    assert (t["out"] == 7.0).all()


@pytest.mark.parametrize("nodes,qh,kvh,dim", [(3, 4, 4, 64), (9, 2, 1, 128), (16, 8, 2, 64),
                                              (16, 8, 2, 128), (70, 4, 2, 128), (128, 4, 2, 64)])
def test_one_long_among_short(tmc, nodes, qh, kvh, dim):
    """One request has nearly all of the steps, the others one or none."""
    cached = [3] * 20 + [24000] + [0] * 20
    f = Forest(15, cached, nodes, qh, kvh, dim, 16, counts=[1 if c < 10 else nodes for c in cached])
    t = f.device()
    f.attend(tmc, t)
    f.check(t, requests=[0, 19, 20, 21, 40])


@pytest.mark.parametrize("nodes,qh,kvh,dim", [(2, 2, 1, 64), (40, 2, 1, 64), (40, 2, 1, 128)])
def test_one_request_one_head(tmc, nodes, qh, kvh, dim):
    """As many pieces as there can be of one (request, kv head)."""
    f = Forest(16, [40000], nodes, qh, kvh, dim, 64)
    t = f.device()
    f.attend(tmc, t)
    f.check(t)


@pytest.mark.parametrize("batch,nodes,dim", [(300, 2, 64), (70, 20, 128)])
def test_many_requests(tmc, batch, nodes, dim):
    rng = random.Random(17)
    cached = [rng.choice([0, 1, 15, 16, 100, 700]) for _ in range(batch)]
    f = Forest(17, cached, nodes, 4, 2, dim, 16, counts=[rng.randint(0, nodes) for _ in cached])
    t = f.device()
    f.attend(tmc, t)
    f.check(t)


@pytest.mark.parametrize("batch,nodes,qh,kvh,dim,most,longest", [
    (40, 4, 16, 4, 128, 300, 1400),    # many pairs, up to 32 vectors: whole, the longest's steps
    (40, 4, 16, 4, 128, 300, 2500),    # shared out
    (2, 8, 8, 2, 64, 500, 700),        # few pairs, whole and shared
    (2, 8, 8, 2, 64, 500, 600),
    (40, 16, 16, 4, 128, 200, 1400),   # one tile of 64, many pairs
    (40, 16, 16, 4, 64, 200, 2000),
    (3, 16, 8, 2, 128, 300, 550),      # few
    (3, 16, 8, 2, 128, 300, 900),
    (3, 25, 8, 1, 128, 200, 3000),     # one tile of 256
    (40, 25, 32, 4, 128, 100, 1400),
    (3, 25, 8, 1, 64, 200, 3000),      # tiles of 64
    (70, 25, 16, 2, 64, 60, 600),      # more tiles than there are counters
    (5, 128, 64, 8, 64, 60, 700),      # tiles of 256 of few pairs
    (5, 128, 64, 8, 128, 60, 700),
    (22, 96, 16, 4, 128, 20, 600),     # tiles of 128
    (22, 96, 16, 4, 64, 20, 600),
    (66, 32, 32, 8, 128, 30, 500),     # tiles of 128, shared and whole
    (66, 32, 32, 8, 128, 30, 200),
    (66, 60, 32, 8, 128, 20, 500),     # tiles of 256 of many pairs
])
def test_ways_of_sharing(tmc, batch, nodes, qh, kvh, dim, most, longest):
    rng = random.Random(19)
    cached = [rng.randint(0, most) for _ in range(batch)]
    at = batch // 2
    cached[at] = longest - nodes
    f = Forest(19, cached, nodes, qh, kvh, dim, 16)
    t = f.device()
    f.attend(tmc, t)
    f.check(t, requests=sorted({0, at, batch - 1, rng.randrange(batch)}))


@pytest.mark.parametrize("nodes", [6, 16, 70])
def test_two_at_once(tmc, nodes):
    """On two streams with a workspace each, neither waiting for the other."""
    pair = [Forest(20 + i, [900 * (i + 1), 20, 3000], nodes, 8, 2, 128, 16) for i in range(2)]
    ts, spaces = [f.device() for f in pair], [f.workspace(tmc) for f in pair]
    streams = [torch.cuda.Stream() for _ in pair]
    torch.cuda.synchronize()
    for _ in range(6):
        for f, t, space, stream in zip(pair, ts, spaces, streams):
            f.attend(tmc, t, workspace=space, stream=stream)
    torch.cuda.synchronize()
    for f, t in zip(pair, ts):
        f.check(t)
