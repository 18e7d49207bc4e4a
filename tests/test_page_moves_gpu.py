"""Page moves and rebuilt block tables: bit copies, so every check is exact."""
import random

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "GPU tests need a GPU"
    return t


def fill(torch, dtype, shape, seed):
    """Every bit pattern, NaNs among them."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    size = torch.empty(0, dtype=dtype).element_size()
    raw = torch.randint(0, 256, (*shape[:-1], shape[-1] * size), generator=g, device="cuda",
                        dtype=torch.uint8)
    return raw.view(dtype)


def same(torch, a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("dtype,layers,heads,page,d", [
    ("float16", 3, 8, 16, 128), ("float16", 33, 2, 12, 64), ("float16", 70, 1, 1, 8),
    ("float32", 2, 4, 16, 32), ("bfloat16", 1, 3, 5, 10), ("float16", 2, 3, 7, 5),
    ("float32", 1, 1, 3, 1), ("float16", 1, 32, 256, 128), ("float32", 1, 5, 9, 6),
    ("float16", 130, 2, 3, 8), ("float16", 2, 3, 1100, 8), ("float16", 1, 1, 4096, 256),
    ("bfloat16", 2, 5, 700, 3)])
def test_moves_copy_the_positions(tmc, torch, dtype, layers, heads, page, d):
    dtype = getattr(torch, dtype)
    pages = 23
    keys = [fill(torch, dtype, (pages, heads, page, d), 2 * i) for i in range(layers)]
    values = [fill(torch, dtype, (pages, heads, page, d), 2 * i + 1) for i in range(layers)]
    rng = random.Random(layers * 31 + d)
    moves = []
    for layer in range(layers):
        order = list(range(pages))
        rng.shuffle(order)
        for i in range(rng.randint(0, 7)):
            # one source for several destinations now and then
            moves.append((layer, order[rng.randint(0, 4)], order[5 + i],
                          rng.choice([1, page, rng.randint(1, page)])))
    want = []
    for pools in (keys, values):
        copies = [t.clone() for t in pools]
        for layer, source, target, n in moves:
            copies[layer][target, :, :n] = pools[layer][source, :, :n]
        want.append(copies)
    tmc.move_pages(keys, values, tmc.page_moves(moves, layers, pages, page), heads, page, d)
    for got, expect in zip((keys, values), want):
        for a, b in zip(got, expect):
            assert same(torch, a, b)


@pytest.mark.parametrize("page_pad,head_pad,offset", [(8, 16, 0), (0, 8, 8), (3, 1, 1), (2, 2, 2)])
def test_moves_in_strided_pools(tmc, torch, page_pad, head_pad, offset):
    """Strides wider than the pages and pools that start off a 16-byte
    boundary; what lies between the pages is left alone."""
    pages, heads, page, d = 9, 3, 4, 16
    head_stride = page * d + head_pad
    page_stride = heads * head_stride + page_pad
    raw = [fill(torch, torch.float16, (pages * page_stride + offset,), s) for s in (1, 2)]
    pools = [t[offset:] for t in raw]
    want = [t.clone() for t in raw]
    moves = [(0, 1, 7, 3), (0, 2, 8, 4), (0, 1, 0, 1)]
    for t in want:
        for _, source, target, n in moves:
            for h in range(heads):
                a, b = (offset + i * page_stride + h * head_stride for i in (source, target))
                t[b:b + n * d] = t[a:a + n * d].clone()
    tmc.move_pages(pools[:1], pools[1:], tmc.page_moves(moves, 1, pages, page), heads, page, d,
                   page_stride=page_stride, head_stride=head_stride)
    for a, b in zip(raw, want):
        assert same(torch, a, b)


def test_bad_moves_copy_nothing(tmc, torch):
    """A device list with moves that name no page, no pool or no positions."""
    pages, heads, page, d = 6, 2, 4, 8
    k, v = (fill(torch, torch.float16, (pages, heads, page, d), s) for s in (3, 4))
    kw, vw = k.clone(), v.clone()
    for t in (kw, vw):
        t[5] = t[0]
    big = 2 ** 31 - 1
    moves = torch.tensor([(0, -1, 1, 4), (0, 6, 1, 4), (0, 1, 6, 4), (0, 1, -1, 4), (1, 1, 2, 4),
                          (-1, 1, 2, 4), (0, 1, 2, 0), (0, 1, 2, 5), (0, 1, 2, -3), (0, 3, 3, 4),
                          (big, 1, 2, 4), (0, big, 2, 4), (0, 1, big, 4), (0, 1, 2, big),
                          (-big - 1, 1, 2, 4), (0, -big - 1, 2, 4), (0, 0, 5, 4)],
                         dtype=torch.int32, device="cuda")
    tmc.move_pages([k], [v], moves, heads, page, d)
    assert same(torch, k, kw) and same(torch, v, vw)
    tmc.move_pages([k], [v], moves[:0], heads, page, d)
    tmc.move_pages([k], [v], tmc.page_moves([], 1, pages, page), heads, page, d)
    assert same(torch, k, kw)


def test_moves_past_4_gib(tmc, torch):
    stride, page, d = 1 << 28, 16, 128
    k, v = (torch.empty(10 * stride, dtype=torch.float16, device="cuda") for _ in range(2))
    rows = []
    for s, pool in enumerate((k, v)):
        rows.append(fill(torch, torch.float16, (page * d,), s))
        pool[stride:stride + page * d] = rows[-1]
        pool[9 * stride:9 * stride + page * d] = 0
    tmc.move_pages([k], [v], tmc.page_moves([(0, 1, 9, page)], 1, 10, page), 1, page, d,
                   page_stride=stride, head_stride=page * d)
    for row, pool in zip(rows, (k, v)):
        assert same(torch, pool[9 * stride:9 * stride + page * d], row)


def plain_tables(tables, parents, remap, slots, tails, pages):
    out = []
    rows = range(len(tables[0])) if parents is None else range(len(parents))
    for layer, table in enumerate(tables):
        new = []
        for r in rows:
            parent = r if parents is None else parents[r]
            row = list(table[parent]) if 0 <= parent < len(table) else [-1] * len(table[0])
            if remap is not None:
                row = [remap[layer][p] if 0 <= p < pages else p for p in row]
            if slots is not None and 0 <= slots[r] < len(row):
                row[slots[r]] = tails[layer][r]
            new.append(row)
        out.append(new)
    return out


@pytest.mark.parametrize("layers,table_rows,rows,max_pages,pages", [
    (1, 1, 1, 1, 1), (32, 16, 16, 37, 300), (3, 5, 64, 9, 40), (2, 64, 3, 513, 2000)])
@pytest.mark.parametrize("use", ["parents", "remap", "tails", "all"])
def test_tables_follow(tmc, torch, layers, table_rows, rows, max_pages, pages, use):
    rng = random.Random(rows * 7 + max_pages)
    every = use == "all"
    if use in ("remap", "tails"):
        rows = table_rows
    entry = lambda: rng.choice([-1, -5, pages, pages + 7, 2 ** 31 - 1] + list(range(pages)) * 3)  # noqa: E731
    tables = [[[entry() for _ in range(max_pages)] for _ in range(table_rows)] for _ in range(layers)]
    parents = ([rng.choice([-1, table_rows, *range(table_rows)]) for _ in range(rows)]
               if use == "parents" or every else None)
    remap = ([[rng.randrange(pages) for _ in range(pages)] for _ in range(layers)]
             if use == "remap" or every else None)
    slots = tails = None
    if use == "tails" or every:
        slots = [rng.choice([-1, max_pages, rng.randrange(max_pages)]) for _ in range(rows)]
        tails = [[rng.randrange(pages) for _ in range(rows)] for _ in range(layers)]
    i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    source = i32(tables)
    out = torch.full((layers, rows, max_pages), 99, dtype=torch.int32, device="cuda")
    tmc.rebuild_tables(source, out, pages, parents=i32(parents), remap=i32(remap),
                       tail_slots=i32(slots), tails=i32(tails))
    want = plain_tables(tables, parents, remap, slots, tails, pages)
    assert out.tolist() == want
    assert source.tolist() == tables
    if parents is None:  # in place
        tmc.rebuild_tables(source, source, pages, remap=i32(remap), tail_slots=i32(slots),
                           tails=i32(tails))
        assert source.tolist() == want


def test_wrappers_refuse(tmc, torch):
    k = torch.zeros(4, 2, 4, 8, dtype=torch.float16, device="cuda")
    moves = torch.tensor([[0, 1, 2, 4]], dtype=torch.int32, device="cuda")
    for args, text in ((([k], [k, k], moves), "as many"), (([], [], moves), "as many"),
                       (([k.cpu()], [k], moves), "current GPU"), (([k], [k], moves.cpu()), "current GPU"),
                       (([k], [k.float()], moves), "must be"), (([k], [k], moves.long()), "moves must"),
                       (([k], [k], moves[0]), "count, 4"),
                       (([k.double()], [k.double()], moves), "float16, bfloat16")):
        with pytest.raises(RuntimeError, match=text):
            tmc.move_pages(*args, 2, 4, 8)
    tables = torch.zeros(1, 3, 4, dtype=torch.int32, device="cuda")
    for kw, text in ((dict(out=tables[0]), "layers"), (dict(out=tables.long()), "out must"),
                     (dict(out=torch.zeros_like(tables), remap=tables[0, 0]), "remap holds"),
                     (dict(out=torch.zeros_like(tables), parents=tables[0, 0, :2]), "parents holds")):
        with pytest.raises(RuntimeError, match=text):
            tmc.rebuild_tables(tables, pool_pages=8, **kw)
