"""Special values, masks and scores in tree attention, for every tile width and every way in
which a request's steps are put together: by one block, by the last of several, by a launch of
its own."""
import random

import numpy as np
import pytest
import torch

from tree_helpers import Forest

pytestmark = pytest.mark.gpu

# batch, nodes, q heads, kv heads, others' most cached positions, the longest's positions
WAYS = {
    "16 whole": (2, 13, 4, 4, 300, 500),
    "16 shared": (2, 13, 4, 4, 300, 1400),
    "32 whole": (3, 14, 8, 4, 300, 500),
    "32 shared": (3, 14, 8, 4, 300, 1400),
    "64 whole": (2, 30, 8, 4, 200, 500),
    "64 joined": (2, 30, 8, 4, 200, 1400),
    "64 shared": (40, 16, 16, 4, 50, 2500),
    "tiles of 64 joined": (2, 20, 8, 2, 300, 1400),
    "128 whole": (2, 20, 8, 2, 30, 200),
    "128 shared": (22, 96, 16, 4, 20, 500),
    "256 whole": (3, 25, 8, 1, 30, 200),
    "256 shared": (40, 25, 32, 4, 60, 2500),
    "256 joined": (2, 20, 8, 2, 300, 52000),  # (head dim 64: tiles of 64)
}


def forest(seed, way, dim, **more):
    """(forest, requests to look at): the longest, one without a cache, a ragged one."""
    batch, nodes, qh, kvh, most, longest = WAYS[way]
    rng = random.Random(seed)
    cached = [rng.randint(0, most) for _ in range(batch)]
    counts = [rng.randint(1, nodes) for _ in range(batch)]
    cached[0] = 0
    cached[-1], counts[-1] = longest - nodes, nodes
    return Forest(seed, cached, nodes, qh, kvh, dim, 16, counts=counts, **more), \
        sorted({0, batch // 2, batch - 1})


@pytest.fixture(params=list(WAYS))
def way(request):
    return request.param


@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_not_seen_changes_nothing(tmc, way, dim):
    f, requests = forest(61, way, dim)
    for r, c in enumerate(f.cached):
        for j, value in ((3, np.nan), (7, np.inf), (11, -np.inf)):
            if j < f.counts[r]:
                f.k[r][c + j, :, 1] = np.nan
                f.v[r][c + j, :, ::3] = value
    t = f.device()
    f.attend(tmc, t)
    f.check(t, requests=requests)


@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_not_seen_in_v_alone(tmc, way, dim):
    """Scores are numbers everywhere: nodes that do not see the slot have a number too."""
    f, requests = forest(62, way, dim)
    for r, c in enumerate(f.cached):
        for j, value in ((2, np.inf), (5, np.nan), (9, -np.inf)):
            if j < f.counts[r]:
                f.v[r][c + j, :, j::5] = value
    t = f.device()
    f.attend(tmc, t)
    f.check(t, requests=requests)


@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_seen_shows(tmc, way, dim):
    f, requests = forest(63, way, dim)
    for r, c in enumerate(f.cached):
        for d, value in ((5, np.nan), (21, np.inf), (40, -np.inf)):
            f.v[r][0, 0, d] = value
            if f.counts[r] > 1:
                f.v[r][c + 1, -1, d + 3] = value
            if c > 100:
                f.v[r][c - 90, 0, d + 1] = value
    t = f.device()
    f.attend(tmc, t)
    f.check(t, requests=requests)


@pytest.mark.parametrize("dim", [64, 128])
def test_any_masks(tmc, way, dim):
    """Nodes that see nothing of the tree, or (without a cache) nothing at all; later nodes; bits
    behind the count."""
    batch, nodes = WAYS[way][:2]
    rng = random.Random(64)
    sees = [[set() if i % 5 == 0 else {j for j in range(nodes) if rng.random() < 0.3}
             for i in range(nodes)] for _ in range(batch)]
    f, requests = forest(64, way, dim, sees=sees)
    t = f.device()
    f.attend(tmc, t)
    f.check(t, requests=requests)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("falls", [False, True])
def test_maxima_that_lag(tmc, way, dim, falls):
    """Scores that rise (or fall) a little a step, so that the scale in use is behind the maximum
    most of the time; below 2^6 in all, as check() asks."""
    f, requests = forest(65, way, dim)
    f.q[..., 0] = 8.0
    f.q[..., 1:] *= np.float16(0.25)
    for r, x in enumerate(f.k):
        ramp = np.linspace(-20.0, 20.0, len(x)) * np.sqrt(dim) / 8.0
        x[:, :, 0] = (ramp[::-1] if falls else ramp)[:, None]
        x[:, :, 1:] *= np.float16(0.25)
    t = f.device()
    f.attend(tmc, t)
    f.check(t, requests=requests)


@pytest.mark.parametrize("dim", [64, 128])
def test_great_scores(tmc, way, dim):
    """Scores of up to a few thousand: one position takes all the weight."""
    f, requests = forest(66, way, dim)
    f.q *= np.float16(40.0)
    for x in f.k:
        x *= np.float16(8.0)
    t = f.device()
    f.attend(tmc, t)
    got = t["out"].float().cpu().numpy().reshape(f.batch, f.nodes, f.q_heads, f.dim)
    for r in requests:
        want, size = f.exact(r)
        n = f.counts[r]
        # a score of 2^12 is off by 2^-10 in fp32 sums of D products, its weight by as much
        bound = 2.0 ** -10 * np.abs(want) + (2.0 ** -11 + 2.0 ** -8) * size + 2.0 ** -24
        assert (np.abs(got[r, :n] - want) <= bound).all()
        assert (got[r, n:] == 7.0).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_scores_past_their_weights(tmc, way, dim):
    """Scores of 2^24 and more, whose maximum in fp32 is several powers of two off, in requests
    where one visible position alone has the greatest: its V comes out, up to the others' share
    of nothing."""
    f, requests = forest(67, way, dim)
    f.q[:] = np.float16(0.0)
    f.q[..., 0] = np.float16(30000.0)
    for r, x in enumerate(f.k):
        x[:, :, 0] = np.float16(-2000.0) * np.random.default_rng(r).random(x.shape[:2])
        x[0, :, 0] = np.float16(20000.0)  # (cached, or the root, which all nodes see)
    t = f.device()
    f.attend(tmc, t)
    got = t["out"].float().cpu().numpy().reshape(f.batch, f.nodes, f.q_heads, f.dim)
    group = f.q_heads // f.kv_heads
    for r in requests:
        want = np.repeat(f.v[r][0], group, axis=0).astype(np.float64)
        # weights of 1 and 0: V, once rounded more than it is
        assert (np.abs(got[r, :f.counts[r]] - want) <= 2.0 ** -10 * np.abs(want) + 2.0 ** -24).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_same_bits_every_time(tmc, way, dim):
    """Whichever block comes last."""
    f, _ = forest(68, way, dim)
    t = f.device()
    space = f.attend(tmc, t)
    first = t["out"].clone()
    for _ in range(4):
        t["out"].fill_(7.0)
        f.attend(tmc, t, workspace=space)
        assert torch.equal(first, t["out"])
