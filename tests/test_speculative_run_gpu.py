"""Steps of speculative decoding as a program makes them: trees laid out, appended to a
paged cache, attended, a token drawn at every node, the agreeing branch accepted and its
K and V moved up.  The model is a toy whose projections depend on the token alone, so that
what the cache must hold is known to the bit."""
import numpy as np
import pytest
import torch

from sample_helpers import draw

pytestmark = pytest.mark.gpu

VOCAB, NODES, CAPACITY = 6, 13, 160
# node 0 repeats the last token; four below it, two below each of them
PARENTS = [-1, 0, 0, 0, 0] + [1 + i // 2 for i in range(8)]


class Toy:
    def __init__(self, tmc, batch, layers, qh, kvh, dim, page, active, seed):
        self.tmc, self.batch, self.layers, self.active_rows = tmc, batch, layers, active
        self.qh, self.kvh, self.dim, self.page = qh, kvh, dim, page
        self.max_pages = -(-CAPACITY // page)
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.rng = np.random.default_rng(seed)

        def normal(*shape):
            return torch.randn(shape, generator=g, device="cuda")

        self.table = normal(layers, VOCAB, (qh + 2 * kvh) * dim).half()
        self.head = normal(qh * dim, VOCAB) / (qh * dim) ** 0.5 * 6
        angles = torch.rand(CAPACITY + 8, dim // 2, generator=g, device="cuda") * 6
        self.cos, self.sin = angles.cos(), angles.sin()
        self.pages = batch * self.max_pages + 2
        order = torch.argsort(torch.rand(layers, self.pages, generator=g, device="cuda"), dim=1)
        self.tables = order[:, :batch * self.max_pages].reshape(layers, batch, -1).int().contiguous()
        self.active = self.ints([active])
        self.workspace = torch.zeros(
            max(tmc.tree_attention_workspace_bytes(batch, NODES, qh, kvh, dim, CAPACITY),
                tmc.sample_workspace_bytes(batch * NODES, VOCAB)) // 4 + 1, device="cuda")
        self.parents = self.ints(PARENTS).repeat(batch, 1)

    def ints(self, values):
        return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")

    def pools(self):
        shape = (self.pages, self.kvh, self.page, self.dim)
        return [[torch.full(shape, 5.0, dtype=torch.float16, device="cuda")
                 for _ in range(self.layers)] for _ in range(2)]

    def draft(self, last):
        """Tokens of the trees: no two children of a node alike."""
        out = np.empty((self.batch, NODES), np.int64)
        for r in range(self.batch):
            out[r, 0] = last[r]
            out[r, 1:5] = self.rng.permutation(VOCAB)[:4]
            for i in range(4):
                out[r, 5 + 2 * i:7 + 2 * i] = self.rng.permutation(VOCAB)[:2]
        return out

    def buffers(self):
        rows, f16 = self.batch * NODES, torch.float16

        def full(*shape, dtype=torch.int32, value=-9):
            return torch.full(shape, value, dtype=dtype, device="cuda")

        return dict(
            masks=full(self.batch, NODES, 1), depths=full(self.batch, NODES),
            q=full(rows, self.qh * self.dim, dtype=f16, value=0),
            out=full(self.layers, rows, self.qh * self.dim, dtype=f16, value=0),
            chosen=full(self.batch, NODES), share=full(rows, dtype=torch.float32),
            path=full(self.batch, NODES), accepted=full(self.batch),
            emitted=full(self.batch, NODES), longer=full(self.batch))

    def forward(self, k, v, t, qkv, cached):
        """Layout, and every layer's append and attention."""
        tmc, shape = self.tmc, (self.batch, NODES, self.qh, self.kvh, self.dim, self.page,
                                self.max_pages)
        tmc.tree_layout(self.parents, t["masks"], t["depths"])
        for l in range(self.layers):
            tmc.tree_rope_append(qkv[l], self.cos, self.sin, cached, t["depths"], None,
                                 self.tables[l], self.active, t["q"], k[l], v[l], *shape)
            tmc.tree_attention(t["q"], k[l], v[l], cached, t["masks"], None, self.tables[l],
                               self.active, t["out"][l], *shape, self.kvh * self.page * self.dim,
                               self.page * self.dim, workspace=self.workspace)

    def choose(self, k, v, t, logits, uniforms, settings, drafted, cached):
        """Sampling, the accepted branch, and its K and V."""
        tmc = self.tmc
        tmc.sample(logits, uniforms, t["chosen"].view(-1), probability=t["share"],
                   workspace=self.workspace, **settings)
        tmc.tree_accept(drafted, self.parents, t["chosen"], t["path"], t["accepted"], t["emitted"],
                        active=self.active, cached_lengths=cached, new_lengths=t["longer"])
        tmc.tree_keep(k, v, self.tables, cached, t["path"], t["accepted"], self.kvh, self.page,
                      self.dim)

    def logits(self, t):
        return t["out"][-1].float() @ self.head

    def sequential(self, tokens):
        """Pools and rotated queries [layers][batch][position] of these tokens one by one."""
        k, v = self.pools()
        longest = max(map(len, tokens))
        queries = torch.zeros(self.layers, self.batch, longest, self.qh * self.dim,
                              dtype=torch.float16, device="cuda")
        for at in range(longest):
            lengths = self.ints([at + 1 if at < len(row) else 0 for row in tokens])
            ids = torch.tensor([row[at] if at < len(row) else 0 for row in tokens], device="cuda")
            for l in range(self.layers):
                q = torch.zeros(self.batch, self.qh * self.dim, dtype=torch.float16, device="cuda")
                self.tmc.decode_rope_append(
                    self.table[l][ids], self.cos, self.sin, lengths, self.tables[l], self.active, q,
                    k[l], v[l], self.batch, self.qh, self.kvh, self.dim, CAPACITY, self.page,
                    self.max_pages)
                queries[l, :, at] = q
        return k, v, queries

    def rows(self, pool, l, r, n):
        """The first n positions of a request: [n, heads, dim]."""
        at = torch.arange(n, device="cuda")
        page = self.tables[l, r][at // self.page].long()
        return pool[page, :, at % self.page]


def settings_of(toy, rows):
    f32 = dict(dtype=torch.float32, device="cuda")
    return dict(temperature=torch.tensor([0.0 if i % 3 == 0 else 0.9 for i in range(rows)], **f32),
                top_k=toy.ints([4 if i % 2 else 0 for i in range(rows)]),
                top_p=torch.tensor([0.9 if i % 5 else 1.0 for i in range(rows)], **f32),
                min_p=torch.tensor([0.05 if i % 7 == 0 else 0.0 for i in range(rows)], **f32))


@pytest.mark.parametrize("batch,layers,qh,kvh,dim,page,active", [
    (3, 2, 8, 2, 128, 16, 3), (4, 3, 4, 4, 64, 5, 3), (2, 1, 6, 1, 96, 16, 2)])
def test_steps_agree_with_token_by_token(tmc, batch, layers, qh, kvh, dim, page, active):
    toy = Toy(tmc, batch, layers, qh, kvh, dim, page, active, seed=batch * dim)
    k, v = toy.pools()
    rows = batch * NODES
    settings = settings_of(toy, rows)
    columns = {n: c.cpu().numpy() for n, c in settings.items()}
    held = [[] for _ in range(batch)]     # tokens in the cache
    last = toy.rng.integers(0, VOCAB, batch)
    cached = toy.ints([0] * batch)
    seen = []                             # (request, position, layer, output)
    for _ in range(14):
        t = toy.buffers()
        drafted = toy.draft(last)
        ids = torch.as_tensor(drafted, device="cuda").view(-1)
        uniforms = torch.as_tensor(toy.rng.random(rows), dtype=torch.float32).cuda()
        toy.forward(k, v, t, toy.table[:, ids].contiguous(), cached)
        logits = toy.logits(t)
        toy.choose(k, v, t, logits, uniforms, settings, toy.ints(drafted), cached)
        x, u = logits.cpu().numpy(), uniforms.cpu().numpy()
        chosen, out = t["chosen"].cpu().numpy(), t["out"].float().cpu().numpy()
        for i in range(active * NODES):
            token, share = draw(x[i], float(u[i]), **{n: c[i].item() for n, c in columns.items()})
            assert chosen.reshape(-1)[i] == token
            assert abs(float(t["share"][i]) - share) <= 2.0 ** -23 * share + 2.0 ** -34
        path, accepted = t["path"].cpu().numpy(), t["accepted"].cpu().numpy()
        emitted = t["emitted"].cpu().numpy()
        for r in range(batch):
            if r >= active:
                assert accepted[r] == 0
                continue
            node, want = 0, []
            while node >= 0:
                want.append(node)
                node = next((c for c in range(NODES) if PARENTS[c] == node and
                             drafted[r, c] == chosen[r, node]), -1)
            assert accepted[r] == len(want) and path[r, :len(want)].tolist() == want
            assert emitted[r, :len(want)].tolist() == [chosen[r, n] for n in want]
            for s, n in enumerate(want):
                seen += [(r, len(held[r]) + s, l, out[l, r * NODES + n]) for l in range(layers)]
            held[r] += [int(drafted[r, n]) for n in want]
            last[r] = emitted[r, accepted[r] - 1]
        cached = t["longer"]
        assert cached.cpu().tolist()[:active] == [len(h) for h in held[:active]]
    assert max(map(len, held)) > 20  # branches were accepted

    wk, wv, queries = toy.sequential([h or [0] for h in held])
    for l in range(layers):
        for r in range(active):
            n = len(held[r])
            for got, want in ((k, wk), (v, wv)):
                assert torch.equal(toy.rows(got[l], l, r, n), toy.rows(want[l], l, r, n))
    # attention: a weight rounds to 11 bits, and so do sum and output; fp32 adds less than 2^-14
    for r, at, l, got in seen:
        key = toy.rows(wk[l], l, r, at + 1).double().cpu().numpy()
        value = toy.rows(wv[l], l, r, at + 1).double().cpu().numpy()
        q = queries[l, r, at].double().cpu().numpy().reshape(qh, dim)
        for h in range(qh):
            s = key[:, h * kvh // qh] @ q[h] / dim ** 0.5
            w = np.exp(s - s.max())
            w /= w.sum()
            want, size = w @ value[:, h * kvh // qh], w @ np.abs(value[:, h * kvh // qh])
            bound = 2.0 ** -10 * np.abs(want) + (2.0 ** -11 + 2.0 ** -14) * size + 2.0 ** -24
            assert (np.abs(got.reshape(qh, dim)[h] - want) <= bound).all(), (r, at, l, h)


def test_captured_steps_share_a_workspace(tmc):
    """Both halves of a step as graphs, replayed over changing inputs with eager work
    between, against the eager step."""
    toy = Toy(tmc, 3, 2, 8, 2, 128, 16, 3, seed=9)
    rows = toy.batch * NODES
    settings = settings_of(toy, rows)
    k, v = toy.pools()
    t = toy.buffers()
    qkv = torch.zeros(toy.layers, rows, (8 + 4) * 128, dtype=torch.float16, device="cuda")
    logits, uniforms = torch.zeros(rows, VOCAB, device="cuda"), torch.zeros(rows, device="cuda")
    drafted, cached = torch.zeros_like(t["path"]), toy.ints([0] * toy.batch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        toy.forward(k, v, t, qkv, cached)
        toy.choose(k, v, t, logits, uniforms, settings, drafted, cached)
    torch.cuda.current_stream().wait_stream(side)
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        toy.forward(k, v, t, qkv, cached)
    with torch.cuda.graph(second):
        toy.choose(k, v, t, logits, uniforms, settings, drafted, cached)
    for pool in (*k, *v):
        pool.fill_(5.0)
    ek, ev = toy.pools()
    last, lengths = toy.rng.integers(0, VOCAB, toy.batch), toy.ints([0] * toy.batch)
    for _ in range(8):
        tokens = toy.draft(last)
        ids = torch.as_tensor(tokens, device="cuda").view(-1)
        numbers = torch.as_tensor(toy.rng.random(rows), dtype=torch.float32).cuda()
        want = toy.buffers()
        toy.forward(ek, ev, want, toy.table[:, ids].contiguous(), lengths)
        theirs = toy.logits(want)
        toy.choose(ek, ev, want, theirs, numbers, settings, toy.ints(tokens), lengths)
        torch.cuda.synchronize()
        for to, value in ((qkv, toy.table[:, ids]), (cached, lengths), (uniforms, numbers),
                          (drafted, toy.ints(tokens))):
            to.copy_(value)
        first.replay()
        logits.copy_(toy.logits(t))
        second.replay()
        torch.cuda.synchronize()
        for name in want:
            assert torch.equal(t[name], want[name]), name
        for got, ours in ((k, ek), (v, ev)):
            assert all(torch.equal(a, b) for a, b in zip(got, ours))
        lengths = want["longer"].clone()
        emitted, accepted = want["emitted"].cpu().numpy(), want["accepted"].cpu().numpy()
        last = emitted[np.arange(toy.batch), accepted - 1]


def test_keys_refuse(tmc):
    rt = tmc.Runtime()
    shape = "batch=2&nodes=8&q_heads=8&kv_heads=2&head_dim=128&page_size=16&max_pages=4"
    for key, text in (("tree_layout?batch=2", "nodes"), ("tree_rope_append?" + shape, "positions"),
                      ("tree_attention?" + shape + "&dtype=f32", "f16"),
                      ("tree_attention?batch=2&nodes=8", "q_heads"), ("sample?rows=4", "vocab"),
                      ("sample?rows=4&vocab=10&dtype=bf16", "dtype"), ("tree_accept?nodes=4", "batch"),
                      ("tree_keep?batch=2&nodes=8&heads=2&head_dim=128&page_size=16", "max_pages"),
                      ("tree_keep?batch=2&nodes=8&heads=2&head_dim=128&page_size=16&max_pages=4"
                       "&pools=15", "pools")):
        with pytest.raises(RuntimeError, match=text):
            rt.resolve(key)


@pytest.mark.parametrize("counts", [False, True])
def test_a_sequence_of_keys_replays(tmc, counts):
    toy = Toy(tmc, 3, 2, 8, 2, 128, 16, 3, seed=5)
    rows = toy.batch * NODES
    some = toy.ints([NODES, 7, 1]) if counts else None
    settings = settings_of(toy, rows)
    drafted = toy.ints(toy.draft(toy.rng.integers(0, VOCAB, 3)))
    qkv = toy.table[:, drafted.long().view(-1)].contiguous()
    cached = toy.ints([20, 0, 47])
    logits = torch.as_tensor(toy.rng.standard_normal((rows, VOCAB)), dtype=torch.float32).cuda()
    uniforms = torch.as_tensor(toy.rng.random(rows), dtype=torch.float32).cuda()
    k, v = toy.pools()
    for pool in (*k, *v):
        pool.copy_(torch.as_tensor(toy.rng.standard_normal(pool.shape)).half())
    start = [p.clone() for p in (*k, *v)]
    dims = (toy.batch, NODES, 8, 2, 128, 16, toy.max_pages)

    want = toy.buffers()
    tmc.tree_layout(toy.parents, want["masks"], want["depths"], counts=some)
    for l in range(2):
        tmc.tree_rope_append(qkv[l], toy.cos, toy.sin, cached, want["depths"], some, toy.tables[l],
                             toy.active, want["q"], k[l], v[l], *dims)
        tmc.tree_attention(want["q"], k[l], v[l], cached, want["masks"], some, toy.tables[l],
                           toy.active, want["out"][l], *dims, 2 * 16 * 128, 16 * 128,
                           workspace=toy.workspace)
    tmc.sample(logits, uniforms, want["chosen"].view(-1), probability=want["share"],
               workspace=toy.workspace, **settings)
    tmc.tree_accept(drafted, toy.parents, want["chosen"], want["path"], want["accepted"],
                    want["emitted"], counts=some, active=toy.active, cached_lengths=cached,
                    new_lengths=want["longer"])
    tmc.tree_keep(k, v, toy.tables, cached, want["path"], want["accepted"], 2, 16, 128)
    end = [p.clone() for p in (*k, *v)]
    torch.cuda.synchronize()

    rt = tmc.Runtime()
    wrapped, got = [], toy.buffers()

    def bind(t):
        wrapped.append(rt.wrap(t))
        return wrapped[-1]

    b = {n: bind(t) for n, t in got.items() if n != "out"}
    kb, vb = [bind(p) for p in k], [bind(p) for p in v]
    cb, ab, pb = bind(cached), bind(toy.active), bind(toy.parents)
    tail = [bind(some)] if counts else []
    more = "&counts=1" if counts else ""
    shape = f"batch=3&nodes={NODES}"
    dims = f"{shape}&q_heads=8&kv_heads=2&head_dim=128&page_size=16&max_pages={toy.max_pages}"
    steps = [rt.prepare(rt.resolve(f"tree_layout?{shape}{more}"), [pb, *tail],
                        [b["masks"], b["depths"]])]
    for l in range(2):
        table = bind(toy.tables[l])
        steps += [
            rt.prepare(rt.resolve(f"tree_rope_append?{dims}&positions={toy.cos.shape[0]}{more}"),
                       [bind(qkv[l]), bind(toy.cos), bind(toy.sin), cb, b["depths"], table, ab,
                        *tail], [b["q"], kb[l], vb[l]]),
            rt.prepare(rt.resolve(f"tree_attention?{dims}{more}"),
                       [b["q"], kb[l], vb[l], cb, b["masks"], table, ab, *tail],
                       [bind(got["out"][l])])]
    steps += [
        rt.prepare(rt.resolve(f"sample?rows={rows}&vocab={VOCAB}&temperature=1&top_k=1&top_p=1"
                              "&min_p=1"),
                   [bind(logits), bind(uniforms)] + [bind(settings[n]) for n in (
                       "temperature", "top_k", "top_p", "min_p")], [b["chosen"], b["share"]]),
        rt.prepare(rt.resolve(f"tree_accept?{shape}&lengths=1{more}"),
                   [bind(drafted), pb, b["chosen"], ab, *tail, cb],
                   [b["path"], b["accepted"], b["emitted"], b["longer"]]),
        rt.prepare(rt.resolve(f"tree_keep?{shape}&pools=2&heads=2&head_dim=128&page_size=16"
                              f"&max_pages={toy.max_pages}"),
                   [bind(toy.tables), cb, b["path"], b["accepted"]], [*kb, *vb])]
    sequence = rt.sequence(steps)
    for _ in range(4):
        fresh = toy.buffers()
        for name, t in got.items():
            t.copy_(fresh[name])
        for pool, old in zip((*k, *v), start):
            pool.copy_(old)
        torch.cuda.synchronize()
        sequence.run()
        torch.cuda.synchronize()
        for name, t in want.items():
            assert torch.equal(got[name], t), name
        assert all(torch.equal(p, e) for p, e in zip((*k, *v), end))
