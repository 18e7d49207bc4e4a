"""Windowed attention where values are extreme: infinities of V behind small
weights, scores of 2^25 and more, and long tails of small weights.  Each through
the forms of a call: requests that have a block to themselves or share several,
few rows of a chunk, and tiles of 64, 128 and 256 vectors."""
import math

import pytest

from tests.test_window_gpu import attend64, visible

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "GPU tests need a GPU"
    return t


class Stream:
    """One request's cache, its pages in random order, and calls over it."""

    def __init__(self, tmc, torch, positions, kvh, d, page, seed):
        self.tmc, self.torch, self.kvh, self.d, self.page = tmc, torch, kvh, d, page
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.g = g
        self.max_pages = -(-positions // page)
        self.order = torch.randperm(self.max_pages, generator=g, device="cuda")
        self.k = torch.zeros(positions, kvh, d, dtype=torch.float16, device="cuda")
        self.v = torch.zeros_like(self.k)

    def normal(self, *shape):
        torch = self.torch
        return torch.randn(shape, generator=self.g, device="cuda")

    def pools(self):
        torch, n = self.torch, self.max_pages * self.page
        made = []
        for t in (self.k, self.v):
            whole = torch.zeros(n, self.kvh, self.d, dtype=torch.float16, device="cuda")
            whole[:t.shape[0]] = t
            pool = torch.empty(self.max_pages, self.kvh, self.page, self.d, dtype=torch.float16,
                               device="cuda")
            pool[self.order] = whole.reshape(self.max_pages, self.page, self.kvh, self.d).transpose(1, 2)
            made.append(pool)
        return made

    def attend(self, form, q, valid, window, sinks, layout=0):
        """Outputs [rows, heads, d] of the rows q [rows, heads, d] at the lengths `valid`."""
        tmc, torch = self.tmc, self.torch
        k, v = self.pools()
        rows, heads, d = q.shape
        lengths = torch.tensor(valid, dtype=torch.int32, device="cuda")
        table = self.order.to(torch.int32)[None]
        out = torch.full((rows, heads * d), 7.5, dtype=torch.float16, device="cuda")
        geometry = (rows, heads, self.kvh, d, self.page, self.max_pages, self.kvh * self.page * d,
                    self.page * d, window, sinks)
        flat = q.reshape(rows, heads * d).contiguous()
        if form == "decode":
            ws = torch.zeros(tmc.window_attention_workspace_bytes(
                rows, heads, self.kvh, d, self.max_pages * self.page, window, sinks) // 4 + 1,
                device="cuda")
            tmc.window_decode_attention(flat, k, v, lengths, table.repeat(rows, 1), None, out,
                                        *geometry, workspace=ws)
        else:
            active = torch.tensor([rows], dtype=torch.int32, device="cuda")
            tmc.window_prefill_attention(flat, k, v, lengths, table, None, active, out, *geometry)
        return out.reshape(rows, heads, d)


# form, rows, query heads, kv heads, head dim, page, length of the last row, window, sinks
FORMS = [
    ("decode", 3, 8, 2, 128, 16, 250, 200, 4),       # a block a row
    ("decode", 3, 8, 2, 64, 12, 500, 400, 4),
    ("decode", 1, 8, 2, 128, 16, 3000, 2500, 4),     # rows shared by blocks
    ("decode", 2, 6, 2, 64, 16, 5000, 4500, 4),
    ("decode", 40, 16, 8, 128, 16, 300, 200, 4),     # blocks of four waves
    ("decode", 80, 16, 8, 64, 16, 300, 200, 4),      # ... and of one
    ("decode", 3, 8, 2, 80, 16, 250, 200, 4),        # the other head dims
    ("chunk", 3, 8, 2, 128, 16, 300, 200, 4),        # few rows
    ("chunk", 20, 34, 2, 64, 16, 300, 200, 4),
    ("chunk", 700, 8, 2, 128, 16, 2300, 1500, 4),    # tiles of 64
    ("chunk", 700, 6, 2, 64, 12, 3900, 3000, 4),
    ("chunk", 300, 64, 64, 128, 16, 1900, 1500, 4),  # 128
    ("chunk", 300, 64, 64, 64, 16, 3600, 3000, 4),
    ("chunk", 300, 80, 80, 128, 16, 1900, 1500, 4),  # 256
    ("chunk", 300, 240, 80, 64, 16, 2600, 2100, 4),
    ("chunk", 40, 8, 2, 80, 16, 300, 200, 4),
]


def lengths_of(form, rows, last):
    return list(range(last - rows + 1, last + 1)) if form == "chunk" else [last - i for i in range(rows)]


def some(rows):
    return sorted({*range(0, rows, 41), 1 % rows, rows // 2, rows - 1})


@pytest.mark.parametrize("form,rows,qh,kvh,d,page,last,window,sinks", FORMS)
def test_infinite_values_behind_small_weights(tmc, torch, form, rows, qh, kvh, d, page, last, window,
                                              sinks):
    """An infinity of V that a row sees makes its dim infinite however small its
    weight is, down to 2^-120 of the greatest; two of opposite signs make a NaN; the
    other dims keep their values."""
    s = Stream(tmc, torch, last, kvh, d, page, 3 * rows + d)
    group = qh // kvh
    valid = lengths_of(form, rows, last)
    s.v.copy_(s.normal(last, kvh, d))
    # all scores are 0 but those of two positions that every row sees, which lie
    # `gap` of the head below in the exponent of 2
    low = max(n - window for n in valid)
    plus, minus = low + 3, min(valid) - 2
    assert sinks <= low < plus < minus
    s.k[plus, :, 0] = s.k[minus, :, 0] = -8.0
    q = torch.zeros(rows, qh, d, device="cuda")
    gaps = [1.0, 30.0, 41.0, 60.0, 100.0, 120.0]
    for h in range(qh):
        q[:, h, 0] = gaps[h % len(gaps)] * math.sqrt(d) / (8.0 * math.log2(math.e))
    s.v[plus, :, 5], s.v[minus, :, 9] = math.inf, -math.inf
    s.v[plus, :, 11], s.v[minus, :, 11] = math.inf, -math.inf
    q = q.to(torch.float16)
    got = s.attend(form, q, valid, window, sinks)
    assert (got[:, :, 5] == math.inf).all()
    assert (got[:, :, 9] == -math.inf).all()
    assert torch.isnan(got[:, :, 11]).all()
    odd = torch.tensor([5, 9, 11], device="cuda")
    clean = s.v.clone()
    clean[:, :, odd] = 0.0
    for r in some(rows):
        see = torch.tensor(visible(valid[r], window, sinks), device="cuda")
        for kh in {0, kvh - 1}:
            mine = slice(kh * group, (kh + 1) * group)
            o, tolerance = attend64(torch, q[r, mine], s.k[see, kh:kh + 1], clean[see, kh:kh + 1])
            near = (got[r, mine].double() - o).abs() <= tolerance
            near[:, odd] = True
            assert near.all(), r


@pytest.mark.parametrize("scale", [2000.0, 8000.0])
@pytest.mark.parametrize("form,rows,qh,kvh,d,page,last,window,sinks", FORMS)
def test_scores_far_from_zero(tmc, torch, form, rows, qh, kvh, d, page, last, window, sinks, scale):
    """Scores of 2^25 to 2^30, where a rounding of a score in fp32 is several powers
    of two of its weight.  Each query is the key of one of its positions, which
    then takes all the weight: the margin to the next score is far above the error
    of fp32 scores (D 2^-24 of the sum of the products' magnitudes), so the output
    is that position's V, rounded to fp16 already."""
    s = Stream(tmc, torch, last, kvh, d, page, 5 * rows + d)
    group = qh // kvh
    valid = lengths_of(form, rows, last)
    s.k.copy_((s.normal(last, kvh, d) * scale).clamp(-60000.0, 60000.0))
    s.v.copy_(s.normal(last, kvh, d))
    low, high = max(n - window for n in valid), min(valid)
    at = (low + torch.arange(rows * qh, device="cuda") * 7919 % (high - low)).reshape(rows, qh)
    heads = torch.arange(qh, device="cuda") // group
    q = s.k[at, heads]
    got = s.attend(form, q, valid, window, sinks)
    for r in some(rows):
        see = torch.tensor(visible(valid[r], window, sinks), device="cuda")
        for h in {0, qh // 2, qh - 1}:
            kk, qq = s.k[see, heads[h]].double(), q[r, h].double()
            scores = kk @ qq / math.sqrt(d)
            error = d * 2.0 ** -24 * ((kk * qq).abs().sum(-1) / math.sqrt(d)).max()
            two = torch.topk(scores, 2).values
            assert two[0] > 2 ** 24 and two[0] - two[1] > 2 * error + 100
    assert torch.equal(got, s.v[at, heads])


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("form,rows,qh,kvh,d,positions", [
    ("decode", 1, 4, 1, 128, 1 << 20), ("decode", 1, 4, 1, 64, 1 << 20),
    ("decode", 70, 4, 4, 128, 60000), ("chunk", 40, 4, 1, 64, 60000),
    ("chunk", 600, 4, 1, 128, 60000), ("chunk", 600, 4, 1, 64, 60000),
    ("chunk", 520, 32, 32, 128, 30000), ("chunk", 520, 48, 48, 64, 30000)])
def test_long_tails_of_small_weights(tmc, torch, form, rows, qh, kvh, d, positions, first):
    """One position with the greatest weight, at the start or the end, and a tail of
    all the others at 2^-24 to 2^-30 of it, which together weigh up to 2^-8: the
    sum of the weights and the products take the same ones, so a mean of ones is
    one.  Tolerance: half a step of fp16 below one, 2^-12, taken twice, and 2^-24
    for each fp32 addition that follows another: of at most 30000 positions of a
    wave, 7500 in the sum (two lanes a vector, two at a time) and 1900 in the
    products (16 at a time)."""
    page, window = 64, positions
    s = Stream(tmc, torch, positions, kvh, d, page, positions + d)
    s.v.fill_(1.0)
    s.k[0 if first else positions - rows, :, 0] = 8.0
    q = torch.zeros(rows, qh, d, device="cuda")
    gaps = [24.3, 25.6, 28.2, 29.3]
    for h in range(qh):
        q[:, h, 0] = gaps[h % 4] * math.sqrt(d) / (8.0 * math.log2(math.e))
    valid = lengths_of(form, rows, positions)
    got = s.attend(form, q.to(torch.float16), valid, window, 4)
    assert ((got.double() - 1.0).abs() <= 2.0 ** -11 + 9400 * 2.0 ** -24).all()


@pytest.mark.parametrize("form,rows,qh,kvh,d,page,last,window,sinks", FORMS)
def test_nan_and_infinite_operands_stay_where_they_are(tmc, torch, form, rows, qh, kvh, d, page, last,
                                                       window, sinks):
    """A NaN of q makes its head NaN and no other; an infinity of K makes a score
    +inf, and the head NaN, or -inf, and its position weigh nothing, by the sign
    of q; a NaN of V makes its dim NaN alone."""
    s = Stream(tmc, torch, last, kvh, d, page, 7 * rows + d)
    group = qh // kvh
    valid = lengths_of(form, rows, last)
    s.k.copy_(s.normal(last, kvh, d))
    s.v.copy_(s.normal(last, kvh, d))
    low = max(n - window for n in valid)
    odd_k, odd_v = low + 5, low + 9
    assert sinks <= low and odd_v < min(valid)
    s.k[odd_k, :, 1] = math.inf
    s.v[odd_v, :, 7] = math.nan
    q = s.normal(rows, qh, d).to(torch.float16)
    q[:, :, 1] = -1.0
    heads = torch.arange(qh, device="cuda")
    turn = (heads[None] + torch.arange(rows, device="cuda")[:, None]) % 4
    q[:, :, 3] = torch.where(turn == 1, math.nan, q[:, :, 3])
    q[:, :, 1] = torch.where(turn == 2, 1.0, q[:, :, 1])
    got = s.attend(form, q, valid, window, sinks)
    lost = (turn == 1) | (turn == 2)
    assert torch.isnan(got[lost]).all()
    kept = torch.ones(d, dtype=torch.bool, device="cuda")
    kept[7] = False
    assert torch.isnan(got[:, :, 7]).all()
    assert torch.isfinite(got[~lost][:, kept]).all()
    clean = s.v.clone()
    clean[odd_v, :, 7] = 0.0
    for r in some(rows):
        see = torch.tensor([p for p in visible(valid[r], window, sinks) if p != odd_k], device="cuda")
        for kh in {0, kvh - 1}:
            mine = slice(kh * group, (kh + 1) * group)
            o, tolerance = attend64(torch, q[r, mine].nan_to_num(0.0), s.k[see, kh:kh + 1],
                                    clean[see, kh:kh + 1])
            near = (got[r, mine].double() - o).abs() <= tolerance
            assert (near | lost[r, mine, None] | ~kept[None]).all(), r
