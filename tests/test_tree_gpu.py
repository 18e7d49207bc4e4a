"""Trees of drafted tokens: masks and depths, rotation and append, the branch that
the chosen tokens agree with, and its K and V moved up."""
import random

import pytest
import torch

from tree_helpers import ancestors, mask_words, paged, random_parents

pytestmark = pytest.mark.gpu


def i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("nodes", [1, 2, 31, 32, 33, 63, 64, 65, 200, 256])
def test_layout(tmc, nodes):
    rng = random.Random(nodes)
    parents = [random_parents(rng, nodes), [i - 1 for i in range(nodes)],  # a chain
               [0] * nodes,  # a star (and node 0 its own parent)
               [rng.randint(-3, nodes + 2) for _ in range(nodes)],  # anything
               [2 ** 31 - 1 - i for i in range(nodes)], random_parents(rng, nodes)]
    counts = [nodes, nodes, nodes, nodes, nodes, nodes // 2]
    words = (nodes + 31) // 32
    masks = torch.full((6, nodes, words), 5, dtype=torch.int32, device="cuda")
    depths = torch.full((6, nodes), 5, dtype=torch.int32, device="cuda")
    tmc.tree_layout(i32(parents), masks, depths, counts=i32(counts))
    masks, depths = masks.cpu().numpy(), depths.cpu().numpy()
    for r, p in enumerate(parents):
        sees, n = ancestors(p), counts[r]
        assert (masks[r, :n] == mask_words(sees, nodes)[:n]).all()
        assert (depths[r, :n] == [len(s) - 1 for s in sees[:n]]).all()
        assert (masks[r, n:] == 5).all() and (depths[r, n:] == 5).all()


def test_layout_refusals(tmc):
    one = i32([[0] * 4])
    for args in ((one[0], one, one), (one.float(), one, one), (one, one[:, :3], one),
                 (one, one, one.cpu()), (i32([[0] * 257]), i32([0] * 9 * 257), i32([0] * 257))):
        with pytest.raises(tmc.TmcError):
            tmc.tree_layout(*args)


APPENDS = [
    # batch, nodes, q heads, kv heads, dim, page
    (1, 1, 4, 4, 128, 16), (3, 9, 8, 2, 64, 12), (2, 40, 4, 1, 128, 16), (2, 5, 6, 3, 10, 4),
    (4, 7, 2, 2, 6, 1), (1, 256, 2, 1, 8, 16)]


@pytest.mark.parametrize("batch,nodes,qh,kvh,dim,page", APPENDS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_append(tmc, batch, nodes, qh, kvh, dim, page, dtype):
    rng, gen = random.Random(batch), torch.Generator().manual_seed(nodes)
    cached = [rng.randint(0, 90) for _ in range(batch)]
    counts = [nodes] + [rng.randint(0, nodes) for _ in range(batch - 1)]
    parents = [random_parents(rng, nodes) for _ in range(batch)]
    active = max(1, batch - 1)
    tables, pages = paged(rng, [c + nodes for c in cached], page)
    tables[0][(cached[0] + nodes - 1) // page] = -1 if nodes > page else tables[0][-1]
    qkv = torch.randn(batch, nodes, (qh + 2 * kvh) * dim, generator=gen).to(dtype)
    angle = torch.rand(max(cached) + nodes, dim // 2, generator=gen) * 6.28
    pool = (pages, kvh, page, dim)
    k, v = torch.full(pool, 7.0, dtype=dtype), torch.full(pool, 7.0, dtype=dtype)
    q = torch.full((batch, nodes, qh * dim), 7.0, dtype=dtype)
    depths = [[len(s) - 1 for s in ancestors(p)] for p in parents]
    dev = [x.cuda() for x in (q, k, v)]
    tmc.tree_rope_append(qkv.cuda(), angle.cos().cuda(), angle.sin().cuda(), i32(cached),
                         i32(depths), i32(counts), i32(tables), i32([active]), *dev, batch, nodes,
                         qh, kvh, dim, page, len(tables[0]))
    # the same in 64 bits: a rotated value is two products and a sum in fp32 (half a
    # step each, of at most |even| + |odd|), then rounded to its type
    cos, sin = angle.cos().double(), angle.sin().double()
    wq, wk, wv = q.double(), k.double(), v.double()
    size = [torch.zeros_like(x) for x in (wq, wk, wv)]
    for r in range(active):
        for i in range(counts[r]):
            x = qkv[r, i].double().reshape(-1, dim // 2, 2)
            at = cached[r] + depths[r][i]
            y = torch.stack([x[..., 0] * cos[at] - x[..., 1] * sin[at],
                             x[..., 0] * sin[at] + x[..., 1] * cos[at]], -1)
            big = x.abs().sum(-1, keepdim=True).expand_as(x)
            y[qh + kvh:] = x[qh + kvh:]
            y, big = y.reshape(-1, dim), big.reshape(-1, dim)
            wq[r, i], size[0][r, i] = y[:qh].reshape(-1), big[:qh].reshape(-1)
            slot = cached[r] + i
            where = tables[r][slot // page]
            if where >= 0:
                wk[where, :, slot % page] = y[qh:qh + kvh]
                size[1][where, :, slot % page] = big[qh:qh + kvh]
                wv[where, :, slot % page] = y[qh + kvh:]
    half, least = torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0.0
    for got, want, big in zip(dev, (wq, wk, wv), size):
        got = got.double().cpu()
        assert ((got - want).abs() <= half * want.abs() + 2 * 2.0 ** -24 * big + least).all()
    assert torch.equal(dev[2].double().cpu(), wv)


def test_append_has_the_bits_of_a_decode_append(tmc):
    """A tree of one node is one token a request."""
    batch, qh, kvh, dim, page = 5, 8, 2, 128, 16
    rng, gen = random.Random(1), torch.Generator(device="cuda").manual_seed(2)
    cached = [0, 3, 15, 16, 60]
    tables, pages = paged(rng, [64] * batch, page)
    qkv = torch.randn(batch, (qh + 2 * kvh) * dim, generator=gen, device="cuda").half()
    angle = torch.rand(64, dim // 2, generator=gen, device="cuda") * 6.28
    new = lambda: [torch.zeros(s, dtype=torch.float16, device="cuda") for s in (  # noqa: E731
        (batch, qh * dim), (pages, kvh, page, dim), (pages, kvh, page, dim))]
    a, b = new(), new()
    tmc.tree_rope_append(qkv, angle.cos(), angle.sin(), i32(cached), i32([0] * batch), None,
                         i32(tables), None, *a, batch, 1, qh, kvh, dim, page, 4)
    tmc.check(tmc.lib().tmc_decode_rope_append(
        *[tmc._ptr(x) for x in (qkv, angle.cos(), angle.sin(), i32([c + 1 for c in cached]),
                                i32(tables), i32([batch]), *b)],
        tmc.F16, batch, qh, kvh, dim, 64, page, 4, tmc._stream()))
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_append_stays_inside(tmc):
    """Lengths, depths and pages that do not exist store nothing."""
    qh = kvh = 2
    dim, page, nodes = 8, 4, 3
    qkv = torch.ones(6, nodes, 6 * dim, dtype=torch.float16, device="cuda")
    angle = torch.zeros(12, dim // 2, device="cuda")
    q = torch.zeros(6, nodes, qh * dim, dtype=torch.float16, device="cuda")
    k = torch.zeros(3, kvh, page, dim, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    cached = [-1, 7, 2 ** 31 - 2, 0, 0, 0]  # capacity 8: one node of request 1 fits
    depths = [[0, 0, 0]] * 3 + [[-1, 12, 2 ** 31 - 1], [0, 0, 0], [0, 0, 0]]
    tables = [[0, 1]] * 4 + [[-1, -1], [3, 1 << 30]]
    tmc.tree_rope_append(qkv, angle.cos(), angle.sin(), i32(cached), i32(depths), None, i32(tables),
                         None, q, k, v, 6, nodes, qh, kvh, dim, page, 2)
    assert k.sum() == qh * dim and v.sum() == qh * dim and k[1, :, 3].sum() == qh * dim
    assert (q.sum(-1) != 0).cpu().tolist() == [[False] * 3, [True, False, False], [False] * 3,
                                               [False] * 3, [True] * 3, [True] * 3]


def walk(parents, drafted, chosen, count):
    path = [0] if count else []
    while path:
        at = path[-1]
        below = [i for i in range(at + 1, count) if parents[i] == at and drafted[i] == chosen[at]]
        if not below:
            break
        path.append(below[0])
    return path


@pytest.mark.parametrize("nodes", [1, 2, 30, 64, 65, 130, 256])
def test_accept(tmc, nodes):
    rng, batch = random.Random(nodes), 40
    parents = [random_parents(rng, nodes, 3) for _ in range(batch)]
    parents[1] = [i - 1 for i in range(nodes)]
    parents[2] = [rng.randint(-2, nodes + 1) for _ in range(nodes)]
    few = lambda: [[rng.randint(0, 2) for _ in range(nodes)] for _ in range(batch)]  # noqa: E731
    drafted, chosen = few(), few()
    drafted[1], chosen[1] = [5] * nodes, [5] * nodes  # all of the chain
    counts = [rng.randint(0, nodes) if r > 2 else nodes for r in range(batch)]
    cached, active = [rng.randint(0, 1000) for _ in range(batch)], batch - 4
    path, emitted = (i32([[9] * nodes] * batch) for _ in range(2))
    accepted, lengths = i32([9] * batch), i32([9] * batch)
    tmc.tree_accept(i32(drafted), i32(parents), i32(chosen), path, accepted, emitted,
                    counts=i32(counts), active=i32([active]), cached_lengths=i32(cached),
                    new_lengths=lengths)
    want = [walk(parents[r], drafted[r], chosen[r], counts[r] if r < active else 0)
            for r in range(batch)]
    assert max(map(len, want)) == nodes
    assert accepted.tolist() == [len(w) for w in want]
    assert lengths.tolist() == [c + len(w) for c, w in zip(cached, want)]
    assert path.tolist() == [w + [-1] * (nodes - len(w)) for w in want]
    assert emitted.tolist() == [[chosen[r][i] for i in w] + [-1] * (nodes - len(w))
                                for r, w in enumerate(want)]


def test_accept_without_the_optional(tmc):
    path, emitted, accepted = i32([[9, 9, 9]]), i32([[9, 9, 9]]), i32([9])
    tmc.tree_accept(i32([[1, 2, 3]]), i32([[-1, 0, 0]]), i32([[3, 8, 4]]), path, accepted, emitted)
    assert path.tolist() == [[0, 2, -1]] and emitted.tolist() == [[3, 4, -1]]
    assert accepted.tolist() == [2]


@pytest.mark.parametrize("dtype,dim,heads", [
    (torch.float16, 128, 8), (torch.float16, 64, 1), (torch.float16, 5, 3), (torch.bfloat16, 96, 32),
    (torch.float32, 6, 2), (torch.float16, 2, 3)])
@pytest.mark.parametrize("page", [1, 5, 16])
def test_keep(tmc, dtype, dim, heads, page):
    rng = random.Random(dim + page)
    batch, nodes, layers = 7, 70, 3
    cached = [rng.randint(0, 50) for _ in range(batch)]
    paths = []
    for r in range(batch):
        inner = sorted(rng.sample(range(1, nodes), rng.choice([0, 1, 5, 7, 8, 9, 40])))
        paths.append([0] + inner)
    paths[0] = list(range(nodes))  # all in place
    paths[1] = list(range(0, nodes, 2))
    accepted = [len(p) for p in paths]
    accepted[3] = 0
    rows = [p + [-1] * (nodes - len(p)) for p in paths]
    tables, pools = [], 0
    for layer in range(layers):
        t, pools = paged(rng, [c + nodes for c in cached], page)
        tables.append(t)
    gen = torch.Generator().manual_seed(3)
    pool = lambda: torch.randn(pools, heads, page, dim, generator=gen).to(dtype)  # noqa: E731
    keys, values = [pool() for _ in range(layers)], [pool() for _ in range(layers)]
    got_k, got_v = [x.cuda() for x in keys], [x.cuda() for x in values]
    tmc.tree_keep(got_k, got_v, i32(tables), i32(cached), i32(rows), i32(accepted), heads, page, dim)
    for layer in range(layers):
        for want, got in ((keys[layer], got_k[layer]), (values[layer], got_v[layer])):
            old = want.clone()
            for r in range(batch):
                place = lambda i: (tables[layer][r][(cached[r] + i) // page],  # noqa: E731
                                   (cached[r] + i) % page)
                for step, node in enumerate(paths[r][:accepted[r]]):
                    (p0, s0), (p1, s1) = place(node), place(step)
                    want[p1, :, s1] = old[p0, :, s0]
            assert torch.equal(want, got.cpu())


def test_keep_stays_inside(tmc):
    """Lists that do not increase, lengths and pages that do not exist."""
    batch, nodes, heads, dim, page = 8, 6, 1, 8, 4
    pool = torch.arange(16 * page, dtype=torch.float16).reshape(16, 1, page, 1).expand(-1, -1, -1, dim)
    k, v = [pool.contiguous().cuda()], [pool.contiguous().cuda()]
    tables = [[[2 * r, 2 * r + 1, -1] for r in range(batch)]]
    tables[0][6] = [-1, 16, 2 ** 30]
    cached = [0, 0, -3, 9, 2 ** 31 - 3, 0, 0, 1]
    path = [[0, 3, 2, 5, -1, -1], [0, 9, 2, 3, 4, 5], [0, 2, 3, 4, 5, -1], [0, 2, 3, 4, 5, -1],
            [0, 2, 3, 4, 5, -1], [0, -7, 2, 3, 4, 5], [0, 2, 3, 4, 5, -1], [0, 2, 5, -1, -1, -1]]
    accepted = [4, 6, 5, 5, 5, 6, 5, 100]
    tmc.tree_keep(k, v, i32(tables), i32(cached), i32(path), i32(accepted), heads, page, dim)
    want = pool.reshape(16 * page, dim).clone()
    want[1] = 3           # request 0: one step, then the list falls
    begin = 14 * page     # request 7: path 0 2 5, then -1 though 100 are claimed
    want[begin + 2], want[begin + 3] = begin + 3, begin + 6
    for got in (k[0], v[0]):
        assert torch.equal(got.cpu().reshape(16 * page, dim), want)


def test_keep_refusals(tmc):
    k = torch.zeros(4, 2, 4, 8, dtype=torch.float16, device="cuda")
    tables, cached, path, accepted = i32([[[0, 1]]]), i32([1]), i32([[0, 2]]), i32([2])
    good = ([k], [k.clone()], tables, cached, path, accepted, 2, 4, 8)
    tmc.tree_keep(*good)
    for at, bad in ((0, []), (0, [k, k]), (0, [k.double()]), (0, [k.cpu()]), (2, tables[0]),
                    (2, tables.long()), (3, cached.cpu()), (4, path[0]), (5, accepted.float()),
                    (6, 0), (6, 100000), (8, 0)):
        with pytest.raises(tmc.TmcError):
            tmc.tree_keep(*good[:at], bad, *good[at + 1:])


def test_many_pools(tmc):
    """More layers than a launch takes."""
    layers = 131
    k = [torch.arange(4, dtype=torch.float16, device="cuda").reshape(1, 1, 4, 1) + i
         for i in range(layers)]
    v = [x + 1000 for x in k]
    tmc.tree_keep(k, v, i32([[[0]]] * layers), i32([1]), i32([[0, 2, -1]]), i32([2]), 1, 4, 1)
    for i in range(layers):
        assert k[i].flatten().tolist() == [i, i + 1, i + 3, i + 3]
        assert v[i].flatten().tolist() == [1000 + i, 1001 + i, 1003 + i, 1003 + i]


def test_captured(tmc):
    rng, nodes = random.Random(5), 40
    parents = i32([random_parents(rng, nodes) for _ in range(3)])
    drafted, chosen = (i32([[rng.randint(0, 1) for _ in range(nodes)] for _ in range(3)])
                       for _ in range(2))
    masks, depths = i32([[[0, 0]] * nodes] * 3), i32([[0] * nodes] * 3)
    path, emitted, accepted = i32([[0] * nodes] * 3), i32([[0] * nodes] * 3), i32([0] * 3)

    def go():
        tmc.tree_layout(parents, masks, depths)
        tmc.tree_accept(drafted, parents, chosen, path, accepted, emitted)

    go()
    torch.cuda.synchronize()
    outputs = (masks, depths, path, emitted, accepted)
    want = [x.clone() for x in outputs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for _ in range(3):
        for x in outputs:
            x.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        for x, w in zip(outputs, want):
            assert torch.equal(x, w)
