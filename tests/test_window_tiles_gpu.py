"""Windowed attention in chunks whose rows and windows lie far past the bounds from
which a chunk is done token by token: in tiles of 64, 128 and 256 query vectors,
each over pools past 4 GiB, strides wider than the pages, the whole capacity,
rows of several requests, and replays.  Decode beside it where rows are shared by
several blocks.  Tolerances as in test_window_gpu."""
import math

import pytest

from tests.test_window_gpu import Cache, attend64, check_rows, visible

pytestmark = pytest.mark.gpu

# rows, query heads, kv heads: tiles of 64, 128, 256 vectors
WIDTHS = [(560, 8, 2), (560, 32, 32), (560, 96, 48)]


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "GPU tests need a GPU"
    return t


def normal(torch, seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(torch.float16)


def ints(torch, values):
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("rows,qh,kvh", WIDTHS)
@pytest.mark.parametrize("d", [64, 128])
def test_tiles_of_pools_past_4_gib(tmc, torch, rows, qh, kvh, d):
    """Two pages behind the first 4 GiB of pools whose pages lie 512 MiB apart."""
    page = 1024 if d == 128 else 2048
    window, sinks, n, stride = page + 100, 3, 2 * page, 1 << 28
    k, v = (torch.empty(10 * stride, dtype=torch.float16, device="cuda") for _ in range(2))
    kk, vv = normal(torch, 1 + d, n, kvh, d), normal(torch, 2 + d, n, kvh, d)
    for i, at in enumerate((9, 8)):
        for pool, new in ((k, kk), (v, vv)):
            pool[at * stride: at * stride + kvh * page * d].view(kvh, page, d).copy_(
                new[i * page:(i + 1) * page].permute(1, 0, 2))
    q = normal(torch, 3 + d, rows, qh * d)
    out = torch.full((rows, qh * d), 7.5, dtype=torch.float16, device="cuda")
    first = n - rows + 1
    tmc.window_prefill_attention(q, k, v, ints(torch, range(first, n + 1)), ints(torch, [9, 8])[None],
                                 None, ints(torch, [rows]), out, rows, qh, kvh, d, page, 2, stride,
                                 page * d, window, sinks)
    for r in (0, 1, 77, 300, rows - 1):
        index = torch.tensor(visible(first + r, window, sinks), device="cuda")
        o, tolerance = attend64(torch, q[r].reshape(qh, d), kk[index], vv[index])
        assert ((out[r].double().reshape(qh, d) - o).abs() <= tolerance).all(), r


def stream(torch, last, rows, kvh, d, page, window, sinks, **pads):
    """A cache of one request whose rows see [low, last) and the sinks."""
    first = last - rows + 1
    seen = set(range(max(0, first - window), last)) | set(range(sinks))
    return Cache(torch, last + d, [seen], kvh, d, page, -(-last // page), **pads)


@pytest.mark.parametrize("rows,qh,kvh", WIDTHS)
@pytest.mark.parametrize("d,page,head_pad,page_pad", [(128, 16, 3, 5), (64, 12, 1, 0), (64, 32, 0, 7)])
def test_tiles_of_strided_pools(tmc, torch, rows, qh, kvh, d, page, head_pad, page_pad):
    last, window, sinks = 3400, 2300, 9
    cache = stream(torch, last, rows, kvh, d, page, window, sinks, head_pad=head_pad, page_pad=page_pad)
    q = normal(torch, rows + d, rows, qh * d)
    out = torch.full((rows, qh * d), 7.5, dtype=torch.float16, device="cuda")
    valid = list(range(last - rows + 1, last + 1))
    tmc.window_prefill_attention(q, cache.k, cache.v, ints(torch, valid), cache.tables_dev, None,
                                 ints(torch, [rows - 3]), out, rows, qh, kvh, d, page,
                                 cache.max_pages, cache.page_stride, cache.head_stride, window, sinks)
    picked = [0, 63, 64, 255, 256, 400, rows - 4, rows - 3, rows - 1]
    index = torch.tensor(picked, device="cuda")
    check_rows(torch, out[index], cache, q[index],
               [(0, valid[r]) if r < rows - 3 else None for r in picked], qh, d, window, sinks, 7.5)


@pytest.mark.parametrize("rows,qh,kvh", WIDTHS)
@pytest.mark.parametrize("d", [64, 128])
def test_a_full_window_in_tiles_is_plain_attention(tmc, torch, rows, qh, kvh, d):
    """Tiles, and one token a request, with a window of the whole capacity against
    the entry points without one, within both sides' tolerances."""
    last, page = 2500, 16
    cache = stream(torch, last, rows, kvh, d, page, last, 0)
    cache.k.nan_to_num_(0.0), cache.v.nan_to_num_(0.0, 0.0, 0.0)
    q = normal(torch, rows + d, rows, qh * d)
    valid, active = ints(torch, range(last - rows + 1, last + 1)), ints(torch, [rows])
    cap = cache.max_pages * page
    geometry = (qh, kvh, d, page, cache.max_pages, cache.page_stride, cache.head_stride)
    plain, tiled = (torch.zeros(rows, qh * d, dtype=torch.float16, device="cuda") for _ in range(2))
    tmc.prefill_attention(q, cache.k, cache.v, valid, cache.tables_dev, active, plain, rows, *geometry)
    tmc.window_prefill_attention(q, cache.k, cache.v, valid, cache.tables_dev, None, active, tiled,
                                 rows, *geometry, cap, 0)
    few = 5
    one, other = (torch.zeros(few, qh * d, dtype=torch.float16, device="cuda") for _ in range(2))
    tables, count = cache.tables_dev.repeat(few, 1), ints(torch, [few])
    space = lambda need: torch.zeros(need // 4 + 1, device="cuda")  # noqa: E731
    tmc.paged_decode_attention(q[:few], cache.k, cache.v, valid[:few], tables, count, one, few,
                               *geometry, space(tmc.attention_workspace_bytes(few, qh, kvh, d, cap)))
    tmc.window_decode_attention(q[:few], cache.k, cache.v, valid[:few], tables, count, other, few,
                                *geometry, cap, 0,
                                space(tmc.window_attention_workspace_bytes(few, qh, kvh, d, cap, cap, 0)))
    _, kk, vv = cache.kv[0]
    for r in (0, 1, 2, 3, 4, 200, rows - 1):
        n = last - rows + 1 + r
        o, tolerance = attend64(torch, q[r].reshape(qh, d), kk[:n], vv[:n])
        outs = [plain, tiled] + ([one, other] if r < few else [])
        for a in outs:
            assert ((a[r].double().reshape(qh, d) - o).abs() <= tolerance).all(), r


@pytest.mark.parametrize("rows,qh,kvh", WIDTHS)
@pytest.mark.parametrize("d,page", [(128, 16), (64, 12)])
def test_tiles_of_several_requests(tmc, torch, rows, qh, kvh, d, page):
    """Runs of one to hundreds of rows of four requests, in and across tiles, with
    rows that keep their output between them."""
    window, sinks, last = 2300, 2 * page + 1, 2900
    max_pages = -(-last // page)
    runs = [(0, 2400, 1), (1, 30, 70), (2, 2600, 5), (3, 1, 40), (9, 100, 3), (0, 2401, 130), (1, 0, 2),
            (2, 2605, 200), (-1, 50, 1), (3, 2800, 100), (0, 2850, 8)]
    row_table = [t for t, _, n in runs for _ in range(n)]
    valid = [start + i for _, start, n in runs for i in range(n)]
    assert len(valid) == rows
    sees = [set() for _ in range(4)]
    good = [0 <= t < 4 and n >= 1 for t, n in zip(row_table, valid)]
    for t, n, ok in zip(row_table, valid, good):
        if ok:
            sees[t] |= set(range(max(0, n - window), n)) | set(range(min(sinks, n)))
    cache = Cache(torch, rows + d, sees, kvh, d, page, max_pages)
    q = normal(torch, rows + d, rows, qh * d)
    out = torch.full((rows, qh * d), 7.5, dtype=torch.float16, device="cuda")
    tmc.window_prefill_attention(q, cache.k, cache.v, ints(torch, valid), cache.tables_dev,
                                 ints(torch, row_table), ints(torch, [rows]), out, rows, qh, kvh, d,
                                 page, max_pages, cache.page_stride, cache.head_stride, window, sinks)
    edges = [0]
    for _, _, n in runs:
        edges.append(edges[-1] + n)
    picked = sorted({e + i for e in edges for i in (-1, 0) if 0 <= e + i < rows} | {63, 64, 127, 128, 255, 256})
    index = torch.tensor(picked, device="cuda")
    check_rows(torch, out[index], cache, q[index],
               [(row_table[r], valid[r]) if good[r] else None for r in picked], qh, d, window, sinks, 7.5)


@pytest.mark.parametrize("rows,qh,kvh", WIDTHS)
@pytest.mark.parametrize("d", [64, 128])
def test_tiles_replay(tmc, torch, rows, qh, kvh, d):
    """A captured chunk and one in the runtime's sequence, replayed over other
    lengths, give the bits of the eager call each time."""
    page, window, sinks, last = 16, 2300, 4, 3000
    cache = stream(torch, last, rows, kvh, d, page, last, 0)
    q = normal(torch, rows + d, rows, qh * d)
    valid, active = ints(torch, range(last - rows + 1, last + 1)), ints(torch, [rows])
    captured, bound = (torch.zeros(rows, qh * d, dtype=torch.float16, device="cuda") for _ in range(2))
    geometry = (rows, qh, kvh, d, page, cache.max_pages, cache.page_stride, cache.head_stride, window,
                sinks)

    def call(out):
        tmc.window_prefill_attention(q, cache.k, cache.v, valid, cache.tables_dev, None, active, out,
                                     *geometry)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(captured)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(captured)
    rt = tmc.Runtime()
    held = [rt.wrap(t) for t in (q, cache.k, cache.v, valid, cache.tables_dev, active, bound)]
    step = rt.prepare(rt.resolve(f"window_prefill_attention?rows={rows}&q_heads={qh}&kv_heads={kvh}"
                                 f"&head_dim={d}&page_size={page}&max_pages={cache.max_pages}"
                                 f"&window={window}&sinks={sinks}"), held[:6], held[6:])
    sequence = rt.sequence([step])
    seen = []
    for turn in range(4):
        first = last - rows + 1 - 100 * (turn % 3)
        valid.copy_(ints(torch, range(first, first + rows)))
        eager = torch.zeros_like(captured)
        call(eager)
        captured.zero_(), bound.zero_()
        graph.replay()
        torch.cuda.synchronize()
        sequence.run()
        torch.cuda.synchronize()
        for out in (captured, bound):
            assert torch.equal(out.view(torch.int16), eager.view(torch.int16)), turn
        seen.append(eager)
    assert torch.equal(seen[0], seen[3]) and not torch.equal(seen[0], seen[1])


@pytest.mark.parametrize("b,qh,kvh,d,last,window", [
    (3, 8, 2, 128, 3000, 2500), (18, 16, 4, 64, 2000, 1800), (1, 34, 2, 128, 9000, 8000)])
def test_packed_output_of_shared_rows(tmc, torch, b, qh, kvh, d, last, window):
    """Rows that several blocks share, written in the packed order."""
    page, sinks = 16, 4
    lengths = [last - 37 * i for i in range(b)]
    cache = Cache(torch, b + d, [set(visible(n, window, sinks)) for n in lengths], kvh, d, page,
                  -(-last // page))
    q, valid = normal(torch, b + d, b, qh * d), ints(torch, lengths)
    need = tmc.window_attention_workspace_bytes(b, qh, kvh, d, cache.max_pages * page, window, sinks)
    assert need  # rows are shared
    ws = torch.zeros(need // 4 + 1, device="cuda")
    out = torch.zeros(b, qh * d, dtype=torch.float16, device="cuda")
    packed = torch.zeros(tmc.packed_activation_elements(b, qh * d), dtype=torch.float16, device="cuda")
    for target, layout in ((out, 0), (packed, tmc.Y_PACKED)):
        tmc.window_decode_attention(q, cache.k, cache.v, valid, cache.tables_dev, None, target, b, qh,
                                    kvh, d, page, cache.max_pages, cache.page_stride,
                                    cache.head_stride, window, sinks, ws, layout=layout)
    check_rows(torch, out, cache, q, list(enumerate(lengths)), qh, d, window, sinks, 7.5)
    rows = torch.empty_like(out)
    tmc.pack_activations(packed, out=rows, unpack=True, rows=b, cols=qh * d)
    assert torch.equal(rows.view(torch.int16), out.view(torch.int16))


@pytest.mark.parametrize("b,qh,kvh,d,last,window", [(3, 8, 2, 128, 3000, 2500), (20, 8, 8, 64, 300, 200)])
def test_infinite_values_in_packed_output(tmc, torch, b, qh, kvh, d, last, window):
    """A head that is done again, for an infinity of V behind a small weight, goes to
    its place in the packed order too."""
    page, sinks = 16, 0
    lengths = [last - 37 * (i % 3) for i in range(b)]
    cache = Cache(torch, b + d, [set(visible(n, window, sinks)) for n in lengths], kvh, d, page,
                  -(-last // page))
    at = last - 90
    for r in range(b):
        page_id = int(cache.tables[r, at // page])
        for pool, dim, value in ((cache.k, slice(None), 0.0), (cache.k, 0, -8.0), (cache.v, 3, math.inf)):
            pool.view(-1, kvh, page, d)[page_id, :, at % page, dim] = value
    q = normal(torch, b + d, b, qh, d)
    q[:, :, 0] = 60.0 * math.sqrt(d) / (8.0 * math.log2(math.e))  # 2^-60 of a weight at score 0
    q, valid = q.reshape(b, qh * d).contiguous(), ints(torch, lengths)
    # keys of the other positions: nothing in dim 0
    others = cache.k.view(-1, kvh, page, d)
    others[..., 0] = torch.where(others[..., 0] == -8.0, others[..., 0], others[..., 0] * 0.0)
    need = tmc.window_attention_workspace_bytes(b, qh, kvh, d, cache.max_pages * page, window, sinks)
    ws = torch.zeros(need // 4 + 1, device="cuda")
    out = torch.zeros(b, qh * d, dtype=torch.float16, device="cuda")
    packed = torch.zeros(tmc.packed_activation_elements(b, qh * d), dtype=torch.float16, device="cuda")
    for target, layout in ((out, 0), (packed, tmc.Y_PACKED)):
        tmc.window_decode_attention(q, cache.k, cache.v, valid, cache.tables_dev, None, target, b, qh,
                                    kvh, d, page, cache.max_pages, cache.page_stride,
                                    cache.head_stride, window, sinks, ws, layout=layout)
    assert (out.view(b, qh, d)[:, :, 3] == math.inf).all()
    assert torch.isfinite(out.view(b, qh, d)[:, :, 4:]).all()
    rows = torch.empty_like(out)
    tmc.pack_activations(packed, out=rows, unpack=True, rows=b, cols=qh * d)
    assert torch.equal(rows.view(torch.int16), out.view(torch.int16))
