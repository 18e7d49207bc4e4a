"""Windowed attention with sinks over the paged cache (one token a request, and
chunks of prompts) against the formula in 64 bits.

Tolerance, per output element: the fp16 rounding of the result, 2^-11 |o|; the
weights' rounding to fp16 in the matrix product and in the sum, 2^-11 A each
with A = sum w |v| / sum w; the fp32 scores, off by at most
d = D 2^-24 max sum |q_i k_i| / sqrt(D) (one rounding per term of the sum) plus
2^-22 for the exponential, which moves each weight and their sum by that
relative amount, 2 d A; and half the least subnormal, 2^-25."""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "GPU tests need a GPU"
    return t


def visible(valid, window, sinks):
    return [p for p in range(valid) if p >= valid - window or p < sinks]


class Cache:
    """Pools whose every element outside the visible positions is NaN (K) or
    infinite (V); pages in random order; only the pages needed exist."""

    def __init__(self, torch, seed, tables_of, kv_heads, d, page, max_pages, spare=3,
                 head_pad=0, page_pad=0):
        """tables_of: per table row, the set of positions some query sees."""
        self.torch, self.page, self.max_pages, self.kv_heads, self.d = torch, page, max_pages, kv_heads, d
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        need = [sorted({p // page for p in seen}) for seen in tables_of]
        count = sum(map(len, need)) + spare
        self.pages = count
        self.head_stride = page * d + 8 * head_pad
        self.page_stride = kv_heads * self.head_stride + 8 * page_pad
        order = torch.randperm(count, generator=g, device="cuda").tolist()
        self.k = torch.full((count, self.page_stride), math.nan, dtype=torch.float16, device="cuda")
        self.v = torch.full((count, self.page_stride), math.inf, dtype=torch.float16, device="cuda")
        self.tables = torch.full((len(need), max_pages), -1, dtype=torch.int32)
        self.kv = []  # per table row: position -> (k, v) [kv_heads, d] in float64
        for row, (seen, pages) in enumerate(zip(tables_of, need)):
            for i in pages:
                self.tables[row, i] = order.pop()
            seen = sorted(seen)
            n = max(len(seen), 1)
            kk = torch.randn((n, kv_heads, d), generator=g, device="cuda").to(torch.float16)
            vv = torch.randn((n, kv_heads, d), generator=g, device="cuda").to(torch.float16)
            if seen:
                pos = torch.tensor(seen, device="cuda")
                ids = self.tables[row].cuda().long()[pos // page]
                for pool, new in ((self.k, kk), (self.v, vv)):
                    view = pool.as_strided((count, kv_heads, page, d),
                                           (self.page_stride, self.head_stride, d, 1))
                    view[ids, :, pos % page] = new
            self.kv.append((seen, kk, vv))
        self.tables_dev = self.tables.cuda()


def attend64(torch, q, kk, vv):
    """q [heads, d] over kk, vv [positions, kv heads, d]: (o, tolerance)."""
    group, d = q.shape[0] // kk.shape[1], q.shape[1]
    q, kk, vv = q.double(), kk.double(), vv.double()
    kk = kk.repeat_interleave(group, 1)
    vv = vv.repeat_interleave(group, 1)
    s = (q[None] * kk).sum(-1) / math.sqrt(d)  # [positions, heads]
    spread = ((q[None] * kk).abs().sum(-1) / math.sqrt(d)).max().item()
    w = torch.softmax(s, 0)[..., None]
    o, a = (w * vv).sum(0), (w * vv.abs()).sum(0)
    delta = d * 2.0 ** -24 * spread + 2.0 ** -22
    return o, 2.0 ** -11 * o.abs() + 2 * (2.0 ** -11 + delta) * a + 2.0 ** -25


def check_rows(torch, out, cache, q, rows, heads, d, window, sinks, untouched):
    """rows: (table row, valid) per output row, or None where it keeps its fill."""
    for r, item in enumerate(rows):
        if item is None:
            assert torch.equal(out[r], torch.full_like(out[r], untouched)), f"row {r} was written"
            continue
        table_row, valid = item
        seen, kk, vv = cache.kv[table_row]
        at = {p: i for i, p in enumerate(seen)}
        index = torch.tensor([at[p] for p in visible(valid, window, sinks)], device="cuda")
        o, tolerance = attend64(torch, q[r].reshape(heads, d), kk[index], vv[index])
        got = out[r].double().reshape(heads, d)
        worst = ((got - o).abs() / tolerance).max().item()
        assert worst <= 1.0, f"row {r} valid {valid}: {worst:.2f} of the tolerance"


DECODE = [
    # qh, kvh, d, page, window, sinks, lengths
    (4, 4, 128, 16, 64, 4, [1, 2, 63, 64, 65, 68, 69, 200, 1000]),
    (8, 2, 128, 16, 100, 0, [1, 99, 100, 101, 117, 513]),
    (8, 1, 128, 16, 17, 16, [5, 33, 34, 300]),
    (32, 8, 128, 16, 1024, 4, [65, 700, 1024, 1030, 2500, 4096]),
    (32, 32, 128, 16, 256, 1, [300, 17]),
    (16, 1, 128, 64, 333, 7, [1, 64, 400, 1500]),   # 16 query heads a kv head
    (6, 2, 128, 16, 50, 3, [20, 200]),              # 3 query heads a kv head
    (10, 2, 64, 16, 50, 3, [20, 200]),
    (34, 2, 64, 16, 50, 3, [20, 200]),              # 17 of them
    (71, 1, 64, 16, 400, 3, [1, 20, 2000]),         # 71: 15, 15, 15, 15 and 11 at a time
    (48, 2, 128, 16, 1500, 30, [1400, 3000, 129]),  # 24: 12 and 12
    (128, 1, 128, 64, 5000, 4, [6000, 128]),
    (8, 2, 64, 16, 1, 0, [1, 2, 16, 17, 100]),      # a window of one
    (8, 2, 64, 16, 1, 5, [1, 3, 5, 6, 100]),
    (4, 4, 64, 12, 40, 7, [1, 11, 12, 13, 47, 48, 49, 500]),
    (8, 2, 128, 12, 500, 13, [11, 700, 2000]),
    (8, 2, 64, 1, 30, 4, [1, 30, 34, 35, 90]),      # pages of one position
    (8, 4, 128, 256, 300, 40, [255, 256, 257, 800]),
    (8, 2, 128, 48, 100, 100, [50, 150, 210, 700]),
    (8, 2, 64, 5, 33, 2, [9, 100]),
    (4, 2, 16, 16, 40, 4, [1, 50, 200]),
    (4, 2, 32, 20, 40, 4, [1, 50, 200]),
    (4, 2, 80, 16, 40, 4, [1, 50, 200]),
    (4, 1, 256, 16, 40, 4, [1, 50, 200]),
    (4, 1, 8, 16, 40, 4, [1, 50]),
    (8, 2, 128, 16, 10 ** 12, 10 ** 12, [1, 100, 512]),  # a window past any capacity
    (8, 2, 128, 16, 8192, 64, [20000, 8000, 8256]),
    (8, 8, 64, 16, 2048, 200, [5000, 2100, 2300, 12]),
]


@pytest.mark.parametrize("qh,kvh,d,page,window,sinks,lengths", DECODE)
def test_decode_matches_the_formula(tmc, torch, qh, kvh, d, page, window, sinks, lengths):
    cap_pages = -(-max(lengths) // page) + 1
    # rows that keep their output: lengths of 0, below it and past the capacity, and padding
    valid = list(lengths) + [0, -5, cap_pages * page + 1, 2 ** 31 - 1, 7]
    sees = [set(visible(n, window, sinks)) if 1 <= n <= cap_pages * page else set() for n in valid]
    cache = Cache(torch, 7 * len(lengths) + d, sees, kvh, d, page, cap_pages)
    batch, active = len(valid), len(valid) - 1
    q = torch.randn(batch, qh * d, device="cuda").to(torch.float16)
    out = torch.full((batch, qh * d), 7.5, dtype=torch.float16, device="cuda")
    need = tmc.window_attention_workspace_bytes(batch, qh, kvh, d, cap_pages * page, window, sinks)
    ws = torch.zeros(max(1, need // 4), device="cuda")
    args = (q, cache.k, cache.v, torch.tensor(valid, dtype=torch.int32, device="cuda"),
            cache.tables_dev, torch.tensor([active], dtype=torch.int32, device="cuda"))
    geometry = (batch, qh, kvh, d, page, cap_pages, cache.page_stride, cache.head_stride, window,
                sinks, ws)
    tmc.window_decode_attention(*args, out, *geometry)
    rows = list(enumerate(lengths)) + [None] * 5
    check_rows(torch, out, cache, q, rows, qh, d, window, sinks, 7.5)
    # the same bits on the second call, over the workspace the first one left
    again = torch.full_like(out, 7.5)
    tmc.window_decode_attention(*args, again, *geometry)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    # no active count: every row counts, the last one too
    every = torch.full_like(out, 7.5)
    tmc.window_decode_attention(*args[:5], None, every, *geometry)
    check_rows(torch, every, cache, q, rows[:-1] + [(batch - 1, 7)], qh, d, window, sinks, 7.5)


@pytest.mark.parametrize("d,page,group", [(128, 16, 4), (64, 12, 1), (128, 16, 1), (32, 16, 2)])
def test_decode_missing_pages(tmc, torch, d, page, group):
    """A missing or out-of-range page that the token would see leaves its row
    untouched; one between the sinks and the window changes nothing."""
    kvh, window, sinks, n = 2, 5 * page + 3, page + 1, 40 * page - 2
    cap_pages = 40
    seen = set(visible(n, window, sinks))
    cache = Cache(torch, 5, [seen] * 6, kvh, d, page, cap_pages)
    t = cache.tables
    assert t[0, 10] == -1  # passed pages are given back
    t[0, 10], t[0, 11] = 2 ** 31 - 1, cache.pages  # ... whatever their entries hold
    t[1, (n - 1) // page] = -1          # the newest page
    t[2, (n - window) // page] = cache.pages  # the window's oldest page, past the pool
    t[3, sinks // page] = -7            # the last sink's page
    t[4, 0] = 2 ** 31 - 1
    qh = kvh * group
    q = torch.randn(6, qh * d, device="cuda").to(torch.float16)
    out = torch.full((6, qh * d), 7.5, dtype=torch.float16, device="cuda")
    need = tmc.window_attention_workspace_bytes(6, qh, kvh, d, cap_pages * page, window, sinks)
    ws = torch.zeros(max(1, need // 4), device="cuda")
    valid = torch.full((6,), n, dtype=torch.int32, device="cuda")
    for _ in range(2):
        tmc.window_decode_attention(q, cache.k, cache.v, valid, t.cuda(), None, out, 6, qh, kvh, d,
                                    page, cap_pages, cache.page_stride, cache.head_stride, window,
                                    sinks, ws)
        check_rows(torch, out, cache, q, [(0, n), None, None, None, None, (5, n)], qh, d, window,
                   sinks, 7.5)


@pytest.mark.parametrize("d,page,head_pad,page_pad", [(128, 16, 3, 5), (64, 12, 1, 0), (64, 32, 0, 7)])
def test_decode_strides(tmc, torch, d, page, head_pad, page_pad):
    """Strides wider than the pages (K and V rows interleaved with other data)."""
    lengths, kvh, qh, window, sinks = [5, 100, 400], 2, 8, 90, 4
    cache = Cache(torch, 11, [set(visible(n, window, sinks)) for n in lengths], kvh, d, page,
                  -(-400 // page), head_pad=head_pad, page_pad=page_pad)
    q = torch.randn(3, qh * d, device="cuda").to(torch.float16)
    out = torch.full((3, qh * d), 7.5, dtype=torch.float16, device="cuda")
    ws = torch.zeros(max(1, tmc.window_attention_workspace_bytes(
        3, qh, kvh, d, cache.max_pages * page, window, sinks) // 4), device="cuda")
    tmc.window_decode_attention(q, cache.k, cache.v,
                                torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                                cache.tables_dev, None, out, 3, qh, kvh, d, page, cache.max_pages,
                                cache.page_stride, cache.head_stride, window, sinks, ws)
    check_rows(torch, out, cache, q, list(enumerate(lengths)), qh, d, window, sinks, 7.5)


@pytest.mark.parametrize("d,page", [(128, 16), (64, 12), (64, 16)])
def test_pools_past_4_gib(tmc, torch, d, page):
    """Page offsets past 32 bits: two pages lie behind the first 4 GiB."""
    kvh, qh, window, sinks, n = 2, 8, 20, 3, 2 * page
    stride = 1 << 28  # elements: 512 MiB between pages
    pages = 10
    k = torch.empty(pages * stride, dtype=torch.float16, device="cuda")
    v = torch.empty(pages * stride, dtype=torch.float16, device="cuda")
    kk = torch.randn(n, kvh, d, device="cuda").to(torch.float16)
    vv = torch.randn(n, kvh, d, device="cuda").to(torch.float16)
    for i, at in enumerate((9, 8)):
        for pool, new in ((k, kk), (v, vv)):
            part = pool[at * stride: at * stride + kvh * page * d].view(kvh, page, d)
            part.copy_(new[i * page:(i + 1) * page].permute(1, 0, 2))
    tables = torch.tensor([[9, 8]], dtype=torch.int32, device="cuda")
    q = torch.randn(n, qh * d, device="cuda").to(torch.float16)
    ws = torch.zeros(max(1, tmc.window_attention_workspace_bytes(1, qh, kvh, d, n, window, sinks)
                         // 4), device="cuda")
    out = torch.full((n, qh * d), 7.5, dtype=torch.float16, device="cuda")
    lengths = torch.arange(1, n + 1, dtype=torch.int32, device="cuda")
    active = torch.tensor([n], dtype=torch.int32, device="cuda")
    tmc.window_prefill_attention(q, k, v, lengths, tables, None, active, out, n, qh, kvh, d, page,
                                 2, stride, page * d, window, sinks)
    one = torch.full((1, qh * d), 7.5, dtype=torch.float16, device="cuda")
    tmc.window_decode_attention(q[n - 1:], k, v, lengths[n - 1:], tables, None, one, 1, qh, kvh, d,
                                page, 2, stride, page * d, window, sinks, ws)
    for got, r in [(out[r], r) for r in range(n)] + [(one[0], n - 1)]:
        index = torch.tensor(visible(r + 1, window, sinks), device="cuda")
        o, tolerance = attend64(torch, q[r].reshape(qh, d), kk[index], vv[index])
        assert ((got.double().reshape(qh, d) - o).abs() <= tolerance).all()


@pytest.mark.parametrize("d,batch,kvh", [(64, 300, 8), (128, 300, 8), (128, 2100, 1), (128, 70, 8),
                                         (64, 100, 8), (128, 1000, 1), (64, 40, 32), (128, 64, 8),
                                         (64, 40, 8)])
def test_decode_batches_of_many_rows(tmc, torch, d, batch, kvh):
    """Many (request, kv head) rows: blocks of four waves and of one."""
    page, window, sinks, cap_pages = 16, 40, 4, 8
    lengths = [1 + (37 * i) % 128 for i in range(batch)]
    cache = Cache(torch, batch, [set(visible(n, window, sinks)) for n in lengths], kvh, d, page, cap_pages)
    qh = 2 * kvh
    q = torch.randn(batch, qh * d, device="cuda").to(torch.float16)
    out = torch.full((batch, qh * d), 7.5, dtype=torch.float16, device="cuda")
    ws = torch.zeros(max(1, tmc.window_attention_workspace_bytes(batch, qh, kvh, d, 128, window,
                                                                 sinks) // 4), device="cuda")
    valid = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    active = torch.tensor([batch - 1], dtype=torch.int32, device="cuda")
    tmc.window_decode_attention(q, cache.k, cache.v, valid, cache.tables_dev, active, out, batch, qh,
                                kvh, d, page, cap_pages, cache.page_stride, cache.head_stride,
                                window, sinks, ws)
    picked = sorted({*range(0, batch, 13), batch - 2, batch - 1})
    check_rows(torch, out[torch.tensor(picked, device="cuda")], cache,
               q[torch.tensor(picked, device="cuda")],
               [(r, lengths[r]) if r < batch - 1 else None for r in picked], qh, d, window, sinks, 7.5)


@pytest.mark.parametrize("d,batch,kvh,group", [(128, 90, 8, 4), (64, 90, 8, 2), (128, 40, 8, 3),
                                               (64, 60, 8, 1), (128, 45, 6, 20)])
def test_decode_rows_that_keep_their_output(tmc, torch, d, batch, kvh, group):
    """Batches in which blocks hold one wave or four, with rows of no length, of
    one past the capacity, of a missing page, and padding."""
    page, window, sinks, cap_pages = 16, 150, 4, 20
    rng = torch.Generator()
    rng.manual_seed(batch + d)
    valid = torch.randint(1, cap_pages * page + 1, (batch,), generator=rng).tolist()
    for i, r in enumerate(range(0, batch, 7)):
        valid[r] = [0, -3, cap_pages * page + 1, 2 ** 31 - 1][i % 4]
    sees = [set(visible(n, window, sinks)) if 1 <= n <= cap_pages * page else set() for n in valid]
    cache = Cache(torch, 43, sees, kvh, d, page, cap_pages)
    tables, missing = cache.tables.clone(), set()
    for r in range(3, batch, 11):
        if sees[r]:
            tables[r, (valid[r] - 1) // page] = cache.pages  # a page past the pool
            missing.add(r)
    q = torch.randn(batch, kvh * group * d, device="cuda").to(torch.float16)
    out = torch.full((batch, kvh * group * d), 7.5, dtype=torch.float16, device="cuda")
    ws = torch.zeros(tmc.window_attention_workspace_bytes(batch, kvh * group, kvh, d,
                                                          cap_pages * page, window, sinks) // 4 + 1,
                     device="cuda")
    active = batch - 2
    tmc.window_decode_attention(q, cache.k, cache.v,
                                torch.tensor(valid, dtype=torch.int32, device="cuda"), tables.cuda(),
                                torch.tensor([active], dtype=torch.int32, device="cuda"), out, batch,
                                kvh * group, kvh, d, page, cap_pages, cache.page_stride,
                                cache.head_stride, window, sinks, ws)
    rows = [(r, valid[r]) if r < active and sees[r] and r not in missing else None
            for r in range(batch)]
    assert missing and sum(item is None for item in rows) > batch // 7
    check_rows(torch, out, cache, q, rows, kvh * group, d, window, sinks, 7.5)


def test_decode_packed_layout(tmc, torch):
    lengths, kvh, qh, d, page, window, sinks = [5, 100, 400, 77] * 5, 2, 8, 128, 16, 90, 4
    cache = Cache(torch, 13, [set(visible(n, window, sinks)) for n in lengths], kvh, d, page, 25)
    b = len(lengths)
    q = torch.randn(b, qh * d, device="cuda").to(torch.float16)
    valid = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    ws = torch.zeros(max(1, tmc.window_attention_workspace_bytes(b, qh, kvh, d, 400, window, sinks)
                         // 4), device="cuda")
    out = torch.zeros((b, qh * d), dtype=torch.float16, device="cuda")
    packed = torch.zeros(tmc.packed_activation_elements(b, qh * d), dtype=torch.float16, device="cuda")
    for target, layout in ((out, 0), (packed, tmc.Y_PACKED)):
        tmc.window_decode_attention(q, cache.k, cache.v, valid, cache.tables_dev, None, target, b,
                                    qh, kvh, d, page, 25, cache.page_stride, cache.head_stride,
                                    window, sinks, ws, layout=layout)
    rows = torch.empty_like(out)
    tmc.pack_activations(packed, out=rows, unpack=True, rows=b, cols=qh * d)
    assert torch.equal(rows.view(torch.int16), out.view(torch.int16))


def test_decode_infinite_values_stay(tmc, torch):
    """An infinite visible V gives an infinite output in its dim alone, large
    scores and equal ones are followed, and a -inf score weighs nothing."""
    kvh, qh, d, page, n, window = 1, 4, 128, 16, 300, 200
    cache = Cache(torch, 17, [set(visible(n, window, 0))], kvh, d, page, 19)
    _, kk, vv = cache.kv[0]
    ids = cache.tables[0].tolist()
    pos = 250
    cache.v.view(-1, page, d)[ids[pos // page], pos % page, 5] = math.inf
    q = torch.randn(1, qh * d, device="cuda").to(torch.float16)
    q[0, d:2 * d] = 0          # equal scores: the plain mean
    q[0, 2 * d:3 * d] *= 60    # one key takes nearly all
    out = torch.zeros(1, qh * d, dtype=torch.float16, device="cuda")
    ws = torch.zeros(max(1, tmc.window_attention_workspace_bytes(1, qh, kvh, d, 19 * page, window, 0)
                         // 4), device="cuda")
    tmc.window_decode_attention(q, cache.k, cache.v,
                                torch.tensor([n], dtype=torch.int32, device="cuda"),
                                cache.tables_dev, None, out, 1, qh, kvh, d, page, 19,
                                cache.page_stride, cache.head_stride, window, 0, ws)
    got = out.double().reshape(qh, d)
    o, tolerance = attend64(torch, q[0].reshape(qh, d), kk, vv)
    keep = torch.arange(d, device="cuda") != 5
    assert ((got - o).abs() <= tolerance)[:, keep].all()
    for head in (0, 1, 3):
        assert got[head, 5] == math.inf


@pytest.mark.parametrize("qh,kvh,d", [(4, 1, 128), (4, 1, 64), (200, 200, 64), (200, 200, 128),
                                     (100, 100, 64), (100, 100, 128), (60, 60, 64), (60, 60, 128)])
def test_chunk_special_values_stay_with_those_that_see_them(tmc, torch, qh, kvh, d):
    """An infinity in V and a NaN in K change the rows that see their positions
    and no other row of the tile."""
    rows, start, page, window, sinks = 70, 100, 16, 40, 4
    valid = list(range(start + 1, start + rows + 1))
    max_pages = -(-(start + rows) // page)
    cache = Cache(torch, 19, [set().union(*(visible(n, window, sinks) for n in valid))], kvh, d,
                  page, max_pages)
    ids = cache.tables[0].tolist()
    odd_v, odd_k = start + 20, start + 45
    head = kvh - 1
    cache.v.view(-1, kvh, page, d)[ids[odd_v // page], head, odd_v % page, 7] = math.inf
    cache.k.view(-1, kvh, page, d)[ids[odd_k // page], head, odd_k % page, 9] = math.nan
    q = torch.randn(rows, qh * d, device="cuda").to(torch.float16)
    out = torch.full((rows, qh * d), 7.5, dtype=torch.float16, device="cuda")
    tmc.window_prefill_attention(q, cache.k, cache.v,
                                 torch.tensor(valid, dtype=torch.int32, device="cuda"),
                                 cache.tables_dev, None,
                                 torch.tensor([rows], dtype=torch.int32, device="cuda"), out, rows,
                                 qh, kvh, d, page, max_pages, cache.page_stride, cache.head_stride,
                                 window, sinks)
    seen, kk, vv = cache.kv[0]
    at = {p: i for i, p in enumerate(seen)}
    group = qh // kvh
    for r, n in enumerate(valid):
        see = visible(n, window, sinks)
        index = torch.tensor([at[p] for p in see], device="cuda")
        o, tolerance = attend64(torch, q[r].reshape(qh, d), kk[index], vv[index])
        got = out[r].double().reshape(qh, d)
        near = (got - o).abs() <= tolerance
        mine = torch.zeros_like(near)
        if odd_k in see:
            assert torch.isnan(got[head * group:]).all(), r
            mine[head * group:] = True
        elif odd_v in see:
            assert (got[head * group:, 7] == math.inf).all(), r
            mine[head * group:, 7] = True
        assert (near | mine).all(), r


CHUNK = [
    # rows, start, qh, kvh, d, page, window, sinks
    (1, 0, 4, 4, 128, 16, 64, 4),
    (1, 500, 8, 2, 128, 16, 64, 4),
    (3, 0, 8, 2, 64, 16, 2, 1),
    (64, 0, 4, 4, 128, 16, 16, 0),
    (65, 0, 4, 4, 128, 16, 1000, 4),
    (130, 37, 8, 2, 128, 16, 40, 5),
    (200, 300, 8, 8, 128, 16, 128, 16),
    (300, 1000, 8, 1, 128, 16, 257, 33),
    (100, 1000, 32, 2, 128, 16, 100, 4),     # 16 query heads a kv head
    (70, 400, 6, 2, 128, 16, 90, 9),         # 3 of them
    (70, 400, 10, 2, 64, 32, 90, 9),         # 5
    (40, 200, 34, 2, 64, 16, 90, 9),         # 17
    (257, 700, 4, 4, 64, 16, 100, 7),
    (203, 700, 8, 2, 64, 12, 100, 7),
    (150, 90, 4, 2, 128, 12, 77, 20),
    (90, 100, 8, 2, 64, 1, 30, 4),
    (90, 100, 8, 2, 128, 5, 1, 0),           # a window of one
    (60, 2000, 4, 2, 128, 256, 500, 300),
    (33, 100, 4, 2, 32, 16, 40, 4),
    (33, 100, 4, 2, 80, 16, 40, 4),
    (20, 100, 2, 1, 256, 16, 40, 4),
    (512, 1024, 4, 1, 128, 16, 512, 16),
    (129, 64, 4, 4, 128, 64, 10 ** 12, 3),
    (515, 0, 2, 2, 128, 16, 200, 70),
    # many kv heads: the wide tiles
    (70, 100, 192, 192, 128, 16, 50, 4),
    (300, 40, 192, 96, 64, 12, 77, 9),
    (515, 300, 128, 64, 128, 16, 200, 70),
    (130, 0, 600, 200, 64, 16, 60, 0),
    # between them: tiles of 128
    (70, 100, 100, 100, 128, 16, 50, 4),
    (300, 40, 64, 32, 64, 12, 77, 9),
    (200, 300, 80, 80, 128, 16, 200, 70),
    (130, 0, 150, 50, 64, 16, 60, 0),
    (515, 1000, 36, 36, 128, 64, 700, 20),
    (100, 64, 500, 100, 128, 16, 10 ** 12, 3),
]


@pytest.mark.parametrize("rows,start,qh,kvh,d,page,window,sinks", CHUNK)
def test_chunk_matches_the_formula(tmc, torch, rows, start, qh, kvh, d, page, window, sinks):
    active = max(1, rows - 2) if rows > 3 else rows
    valid = list(range(start + 1, start + rows + 1))
    max_pages = -(-(start + rows) // page)
    sees = set().union(*(visible(n, window, sinks) for n in valid[:active]))
    cache = Cache(torch, rows + d, [sees], kvh, d, page, max_pages)
    q = torch.randn(rows, qh * d, device="cuda").to(torch.float16)
    out = torch.full((rows, qh * d), 7.5, dtype=torch.float16, device="cuda")
    tmc.window_prefill_attention(q, cache.k, cache.v,
                                 torch.tensor(valid, dtype=torch.int32, device="cuda"),
                                 cache.tables_dev, None,
                                 torch.tensor([active], dtype=torch.int32, device="cuda"), out,
                                 rows, qh, kvh, d, page, max_pages, cache.page_stride,
                                 cache.head_stride, window, sinks)
    picked = range(rows) if rows <= 130 else sorted({*range(0, rows, 7), rows - 3, rows - 2, rows - 1,
                                                     63, 64, 65, 127, 128})
    expect = [(0, valid[r]) if r < active else None for r in picked]
    index = torch.tensor(list(picked), device="cuda")
    check_rows(torch, out[index], cache, q[index], expect, qh, d, window, sinks, 7.5)


@pytest.mark.parametrize("rows,start,qh,kvh,d,page,window,sinks", [
    (300, 400, 6, 2, 128, 16, 900, 9),        # 3 query heads a kv head
    (600, 400, 10, 2, 64, 32, 90, 9),         # 5
    (350, 200, 34, 2, 64, 16, 290, 9),        # 17
    (300, 1000, 32, 2, 128, 16, 100, 4),      # 16
    (600, 1000, 64, 1, 128, 16, 257, 33),     # 64
    (300, 500, 65, 1, 64, 16, 200, 3),        # 65: past the tiles
    (600, 90, 4, 2, 128, 12, 77, 20),
    (700, 100, 8, 2, 64, 1, 130, 4),          # pages of one position
    (2100, 100, 8, 2, 128, 5, 1, 0),          # a window of one
    (600, 2000, 4, 2, 128, 256, 500, 300),
    (700, 0, 4, 4, 128, 16, 1000, 4),
    (1100, 0, 4, 4, 128, 16, 16, 0),
    (513, 3000, 4, 1, 128, 16, 10 ** 12, 0),
])
def test_chunk_tiles_match_the_formula(tmc, torch, rows, start, qh, kvh, d, page, window, sinks):
    """Chunks long enough for the tiles; some of their rows are checked."""
    n = start + rows
    max_pages = -(-n // page)
    seen = set()
    for valid in range(start + 1, n + 1):
        seen |= set(range(max(0, valid - min(window, n)), valid)) if valid in (start + 1, n) else {valid - 1}
    seen |= set(range(min(sinks, n)))
    cache = Cache(torch, rows + d, [seen], kvh, d, page, max_pages)
    q = torch.randn(rows, qh * d, device="cuda").to(torch.float16)
    out = torch.full((rows, qh * d), 7.5, dtype=torch.float16, device="cuda")
    tmc.window_prefill_attention(q, cache.k, cache.v,
                                 torch.arange(start + 1, n + 1, dtype=torch.int32, device="cuda"),
                                 cache.tables_dev, None,
                                 torch.tensor([rows - 1], dtype=torch.int32, device="cuda"), out,
                                 rows, qh, kvh, d, page, max_pages, cache.page_stride,
                                 cache.head_stride, window, sinks)
    picked = sorted({*range(0, rows, 29), 1, 63, 64, 127, 128, 255, 256, rows - 2, rows - 1})
    index = torch.tensor(picked, device="cuda")
    check_rows(torch, out[index], cache, q[index],
               [(0, start + 1 + r) if r < rows - 1 else None for r in picked], qh, d, window, sinks,
               7.5)


@pytest.mark.parametrize("qh,kvh,d,page", [(4, 4, 128, 16), (8, 2, 64, 12), (8, 1, 128, 16),
                                           (4, 2, 32, 16), (200, 200, 64, 16), (200, 200, 128, 12),
                                           (90, 90, 64, 12), (90, 90, 128, 16),
                                           (16, 16, 128, 16), (48, 16, 64, 12)])
def test_chunk_of_several_requests(tmc, torch, qh, kvh, d, page):
    """Rows of several requests in any packing, with invalid lengths, table rows
    outside the tables, and a request whose window reaches a missing page."""
    window, sinks, max_pages = 3 * page + 1, page + 2, 30
    plan = [(0, list(range(1, 40))), (1, [200]), (2, list(range(300, 390))), (0, [41, 40]),
            (3, [77]), (2, [12, 500 * page, 0, -3, 25]), (9, [5]), (-1, [5]),
            (1, list(range(201, 205))), (4, list(range(9 * page - 2, 9 * page + 3)))]
    row_table = [t for t, ns in plan for _ in ns]
    valid = [n for _, ns in plan for n in ns]
    cap = max_pages * page
    sees = [set() for _ in range(5)]
    for t, n in zip(row_table, valid):
        if 0 <= t < 5 and 1 <= n <= cap:
            sees[t] |= set(visible(n, window, sinks))
    cache = Cache(torch, 3 + d, sees, kvh, d, page, max_pages)
    # request 4's page 5: only its tokens below 9 pages see it (window 3 pages + 1)
    missing = (9 * page - window) // page
    cache.tables[4, missing] = -1
    rows = len(valid)
    q = torch.randn(rows, qh * d, device="cuda").to(torch.float16)
    out = torch.full((rows, qh * d), 7.5, dtype=torch.float16, device="cuda")
    tmc.window_prefill_attention(q, cache.k, cache.v,
                                 torch.tensor(valid, dtype=torch.int32, device="cuda"),
                                 cache.tables.cuda(),
                                 torch.tensor(row_table, dtype=torch.int32, device="cuda"),
                                 torch.tensor([rows], dtype=torch.int32, device="cuda"), out, rows,
                                 qh, kvh, d, page, max_pages, cache.page_stride, cache.head_stride,
                                 window, sinks)
    expect = []
    for t, n in zip(row_table, valid):
        ok = 0 <= t < 5 and 1 <= n <= cap
        ok = ok and not (t == 4 and any(p // page == missing for p in visible(n, window, sinks)))
        expect.append((t, n) if ok else None)
    assert any(e is None for e in expect[-5:]) and any(e for e in expect[-5:])
    check_rows(torch, out, cache, q, expect, qh, d, window, sinks, 7.5)


def test_full_window_is_plain_attention(tmc, torch):
    """With a window of the whole capacity both forms agree with the
    unwindowed entry points within both sides' tolerances."""
    rows, qh, kvh, d, page, start = 48, 8, 2, 128, 16, 100
    n = start + rows
    max_pages = -(-n // page)
    cache = Cache(torch, 23, [set(range(n))], kvh, d, page, max_pages)
    cache.k.nan_to_num_(0.0), cache.v.nan_to_num_(0.0, 0.0, 0.0)
    q = torch.randn(rows, qh * d, device="cuda").to(torch.float16)
    valid = torch.arange(start + 1, n + 1, dtype=torch.int32, device="cuda")
    active = torch.tensor([rows], dtype=torch.int32, device="cuda")
    a, b = (torch.zeros((rows, qh * d), dtype=torch.float16, device="cuda") for _ in range(2))
    geometry = (rows, qh, kvh, d, page, max_pages, cache.page_stride, cache.head_stride)
    tmc.prefill_attention(q, cache.k, cache.v, valid, cache.tables_dev, active, a, *geometry)
    tmc.window_prefill_attention(q, cache.k, cache.v, valid, cache.tables_dev, None, active, b,
                                 *geometry, max_pages * page, 0)
    _, kk, vv = cache.kv[0]
    for r in range(rows):
        _, tolerance = attend64(torch, q[r].reshape(qh, d), kk[:start + r + 1], vv[:start + r + 1])
        assert ((a[r] - b[r]).double().abs().reshape(qh, d) <= 2 * tolerance).all()


def test_graph_replays_and_streams(tmc, torch):
    """A captured decode step, replayed with eager work of the same kind and
    other lengths in between, gives the eager bits each time; so does a call on
    another stream."""
    kvh, qh, d, page, window, sinks, max_pages, b = 2, 8, 128, 16, 120, 4, 40, 5
    lengths = [[5, 100, 300, 640, 1], [640, 6, 101, 17, 301], [130, 120, 119, 121, 500]]
    sees = [set(range(640))] * b
    cache = Cache(torch, 29, sees, kvh, d, page, max_pages)
    q = torch.randn(b, qh * d, device="cuda").to(torch.float16)
    need = tmc.window_attention_workspace_bytes(b, qh, kvh, d, max_pages * page, window, sinks)
    ws, other = (torch.zeros(max(1, need // 4), device="cuda") for _ in range(2))
    valid = torch.tensor(lengths[0], dtype=torch.int32, device="cuda")
    out = torch.zeros(b, qh * d, dtype=torch.float16, device="cuda")

    def call(target, workspace, n, stream=None):
        tmc.window_decode_attention(q, cache.k, cache.v, n, cache.tables_dev, None, target, b, qh,
                                    kvh, d, page, max_pages, cache.page_stride, cache.head_stride,
                                    window, sinks, workspace, stream=stream)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(out, ws, valid)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out, ws, valid)
    for step in range(6):
        now = torch.tensor(lengths[step % 3], dtype=torch.int32, device="cuda")
        eager = torch.zeros_like(out)
        call(eager, other, now)
        valid.copy_(now)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), eager.view(torch.int16)), step
        away = torch.zeros_like(out)
        side.wait_stream(torch.cuda.current_stream())
        call(away, other, now, stream=side)
        side.synchronize()
        assert torch.equal(away.view(torch.int16), eager.view(torch.int16)), step


def test_two_streams_at_once(tmc, torch):
    """Calls that overlap, each with a workspace of its own and both over one cache."""
    b, qh, kvh, d, page, window, sinks, length = 4, 16, 4, 128, 16, 1500, 4, 2000
    pages = -(-length // page)
    cache = Cache(torch, 37, [set(range(length))] * b, kvh, d, page, pages)
    valid = torch.tensor([length, 1700, 3, 900], dtype=torch.int32, device="cuda")
    need = tmc.window_attention_workspace_bytes(b, qh, kvh, d, pages * page, window, sinks)
    assert need
    streams = [torch.cuda.Stream() for _ in range(2)]
    queries = [torch.randn(b, qh * d, device="cuda").to(torch.float16) for _ in range(2)]
    spaces = [torch.zeros(need // 4 + 1, device="cuda") for _ in range(2)]

    def call(i, out, stream=None):
        tmc.window_decode_attention(queries[i], cache.k, cache.v, valid, cache.tables_dev, None,
                                    out, b, qh, kvh, d, page, pages, cache.page_stride,
                                    cache.head_stride, window, sinks, spaces[i], stream=stream)

    want = [torch.zeros(b, qh * d, dtype=torch.float16, device="cuda") for _ in range(2)]
    for i in range(2):
        call(i, want[i])
    outs = [[torch.zeros_like(want[0]) for _ in range(30)] for _ in range(2)]
    torch.cuda.synchronize()
    for n in range(30):
        for i in range(2):
            call(i, outs[i][n], streams[i])
    torch.cuda.synchronize()
    for i in range(2):
        for out in outs[i]:
            assert torch.equal(out.view(torch.int16), want[i].view(torch.int16))


def test_one_workspace_for_attention_and_scores(tmc, torch):
    """Launches of several shapes and of tmc_logprobs use one workspace in turn,
    eagerly and in two captured graphs that share it."""
    # batch, heads, kv heads, dim, length, window; the last three share no row
    shapes = [(1, 8, 2, 128, 900, 600), (3, 4, 4, 128, 2000, 600), (6, 40, 1, 64, 3000, 2500),
              (16, 8, 8, 64, 1500, 1400), (40, 8, 8, 64, 1500, 1400), (6, 40, 1, 64, 700, 600),
              (40, 8, 8, 64, 300, 600)]
    page, sinks = 16, 4
    vocab, top = 20000, 5
    need = [tmc.logprobs_workspace_bytes(2, vocab, top)]
    calls = []
    for i, (b, qh, kvh, d, length, window) in enumerate(shapes):
        pages = -(-length // page)
        cache = Cache(torch, 31 + i, [set(range(length))] * b, kvh, d, page, pages)
        need.append(tmc.window_attention_workspace_bytes(b, qh, kvh, d, pages * page, window, sinks))
        q = torch.randn(b, qh * d, device="cuda").to(torch.float16)
        valid = torch.full((b,), length, dtype=torch.int32, device="cuda")

        def attend(out, ws, q=q, cache=cache, valid=valid, pages=pages, shape=shapes[i]):
            b, qh, kvh, d, _, window = shape
            tmc.window_decode_attention(q, cache.k, cache.v, valid, cache.tables_dev, None, out, b,
                                        qh, kvh, d, page, pages, cache.page_stride,
                                        cache.head_stride, window, sinks, ws)
        calls.append((attend, q.shape))
    assert all(need[:5])
    logits = torch.randn(2, vocab, device="cuda")
    tokens = torch.tensor([5, vocab - 1], dtype=torch.int32, device="cuda")

    best = torch.empty(2, top, dtype=torch.int32, device="cuda")
    best_lp = torch.empty(2, top, device="cuda")

    def score(out, ws):
        tmc.logprobs(logits, tokens, out[0], out[1], best, best_lp, ws)

    def all_of_them(outs, lp, ws):
        for (attend, _), out in zip(calls, outs):
            attend(out, ws)
            score(lp, ws)

    def outputs():
        return ([torch.zeros(shape, dtype=torch.float16, device="cuda") for _, shape in calls],
                torch.zeros(2, 2, device="cuda"))

    want, want_lp = outputs()
    for (attend, _), out, n in zip(calls, want, need[1:]):
        attend(out, torch.zeros(n // 4 + 1, device="cuda"))  # each on a workspace of its own
    score(want_lp, torch.zeros(need[0] // 4 + 1, device="cuda"))
    ws = torch.zeros(max(need) // 4 + 1, device="cuda")
    graphs, results = [], []
    for _ in range(2):
        outs, lp = outputs()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            all_of_them(outs, lp, ws)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            all_of_them(outs, lp, ws)
        graphs.append(graph)
        results.append((outs, lp))
    for _ in range(3):
        for graph, (outs, lp) in zip(graphs, results):
            for t in (*outs, lp):
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip((*outs, lp), (*want, want_lp)):
                assert torch.equal(a, b)
        outs, lp = outputs()
        all_of_them(outs, lp, ws)
        torch.cuda.synchronize()
        for a, b in zip((*outs, lp), (*want, want_lp)):
            assert torch.equal(a, b)


def test_wrappers_refuse(tmc, torch):
    kvh, qh, d, page, max_pages = 2, 8, 128, 16, 4
    k = torch.zeros(8, kvh, page, d, dtype=torch.float16, device="cuda")
    q = torch.zeros(2, qh * d, dtype=torch.float16, device="cuda")
    out, valid = torch.zeros_like(q), torch.ones(2, dtype=torch.int32, device="cuda")
    tables = torch.zeros(2, max_pages, dtype=torch.int32, device="cuda")
    ws = torch.zeros(1 << 20, device="cuda")

    def call(**change):
        a = dict(q=q, k=k, v=k, valid=valid, tables=tables, out=out, batch=2, window=8, pool=None,
                 workspace=ws)
        a.update(change)
        tmc.window_decode_attention(a["q"], a["k"], a["v"], a["valid"], a["tables"], None, a["out"],
                                    a["batch"], qh, kvh, d, page, max_pages, kvh * page * d,
                                    page * d, a["window"], 2, a["workspace"], pool_pages=a["pool"])

    call()
    for change, text in ((dict(q=q.cpu()), "current GPU"), (dict(tables=tables.cpu()), "current GPU"),
                         (dict(q=q.float()), "q must be"), (dict(valid=valid.long()), "valid_lengths"),
                         (dict(batch=3), "elements"), (dict(out=out[:1]), "out holds"),
                         (dict(tables=tables[:, :2].contiguous()), "tables holds"),
                         (dict(window=0), "window must be at least 1"),
                         (dict(q=torch.zeros(qh * d, 2, dtype=torch.float16, device="cuda").t()),
                          "contiguous"), (dict(pool=9), "pools hold 8")):
        with pytest.raises(RuntimeError, match=text):
            call(**change)
