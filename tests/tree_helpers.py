"""Trees of drafted tokens and a paged cache for the speculative-decoding tests,
with plain 64-bit forms of the operators."""
import math
import random

import numpy as np
import torch

NAN = float("nan")


def random_parents(rng, nodes, reach=6):
    """Parents of one tree: node 0 a root, the others below a node shortly before."""
    return [-1] + [rng.randint(max(0, i - reach), i - 1) for i in range(1, nodes)]


def ancestors(parents):
    """Every node's ancestors and itself, as sets."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if 0 <= p < i else set()) | {i})
    return out


def mask_words(sees, nodes):
    words = (nodes + 31) // 32
    out = np.zeros((len(sees), words), np.uint32)
    for i, s in enumerate(sees):
        for j in s:
            out[i, j >> 5] |= np.uint32(1 << (j & 31))
    return out.view(np.int32)


def paged(rng, lengths, page, spare=3):
    """(tables [rows][max_pages] with -1 behind, pages): so many positions a row on
    pages in random order, `spare` pages in nobody's table."""
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + spare
    order = rng.sample(range(pages), pages)
    width = max(1, max(need))
    return [[order.pop() for _ in range(n)] + [-1] * (width - n) for n in need], pages


class Forest:
    """A batch of requests with a cache, a tree each and everything that the tree
    operators take.  Places of the pools that no position of a request uses hold
    NaN."""

    def __init__(self, seed, cached, nodes, q_heads, kv_heads, dim, page, counts=None,
                 active=None, gap=(0, 0), sees=None):
        rng, gen = random.Random(seed), np.random.default_rng(seed)
        self.cached, self.nodes, self.batch = cached, nodes, len(cached)
        self.q_heads, self.kv_heads, self.dim, self.page = q_heads, kv_heads, dim, page
        self.counts = counts or [nodes] * self.batch
        self.active = self.batch if active is None else active
        self.parents = [random_parents(rng, nodes) for _ in cached]
        self.sees = sees or [ancestors(p) for p in self.parents]
        self.tables, self.pages = paged(rng, [c + nodes for c in cached], page)
        self.max_pages = len(self.tables[0])
        self.head_stride = page * dim + gap[0]
        self.page_stride = kv_heads * self.head_stride + gap[1]
        # [batch][position][kv head][dim]
        self.k = [gen.standard_normal((c + nodes, kv_heads, dim)).astype(np.float16) for c in cached]
        self.v = [gen.standard_normal((c + nodes, kv_heads, dim)).astype(np.float16) for c in cached]
        self.q = gen.standard_normal((self.batch, nodes, q_heads, dim)).astype(np.float16)

    def pool(self, rows):
        flat = np.full(self.pages * self.page_stride, NAN, np.float16)
        for r, x in enumerate(rows):
            for pos in range(len(x)):
                at = (self.tables[r][pos // self.page] * self.page_stride
                      + pos % self.page * self.dim)
                for h in range(self.kv_heads):
                    flat[at + h * self.head_stride:at + h * self.head_stride + self.dim] = x[pos, h]
        return torch.from_numpy(flat).cuda()

    def device(self):
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        masks = np.stack([mask_words(s, self.nodes) for s in self.sees])
        return dict(q=torch.from_numpy(self.q).cuda(), k=self.pool(self.k), v=self.pool(self.v),
                    cached=i32(self.cached), counts=i32(self.counts), tables=i32(self.tables),
                    masks=torch.from_numpy(masks).cuda(), active=i32([self.active]),
                    out=torch.full((self.batch, self.nodes, self.q_heads * self.dim), 7.0,
                                   dtype=torch.float16, device="cuda"))

    def attend(self, tmc, t, workspace=None, stream=None, counts=True, active=True, **more):
        geometry = (self.batch, self.nodes, self.q_heads, self.kv_heads, self.dim, self.page,
                    self.max_pages, self.page_stride, self.head_stride)
        if workspace is None:
            workspace = self.workspace(tmc)
        tmc.tree_attention(t["q"], t["k"], t["v"], t["cached"], t["masks"],
                           t["counts"] if counts else None, t["tables"],
                           t["active"] if active else None, t["out"], *geometry,
                           workspace=workspace, stream=stream, **more)
        return workspace

    def workspace(self, tmc):
        size = tmc.tree_attention_workspace_bytes(self.batch, self.nodes, self.q_heads,
                                                  self.kv_heads, self.dim,
                                                  self.page * self.max_pages)
        return torch.zeros(max(4, size // 4 + 1), device="cuda")

    def exact(self, r):
        """(out, mean |v|) of request r in 64 bits, [count][q heads][dim]."""
        n, c, group = self.counts[r], self.cached[r], self.q_heads // self.kv_heads
        end = c + n
        see = np.zeros((n, end), bool)
        see[:, :c] = True
        for i in range(n):
            for j in self.sees[r][i]:
                if j < n:
                    see[i, c + j] = True
        out = np.zeros((n, self.q_heads, self.dim))
        size = np.zeros((n, self.q_heads, self.dim))
        for h in range(self.q_heads):
            k, v = (x[r][:end, h // group].astype(np.float64) for x in (self.k, self.v))
            with np.errstate(all="ignore"):
                s = self.q[r, :n, h].astype(np.float64) @ k.T / math.sqrt(self.dim)
            for i in range(n):
                at = np.flatnonzero(see[i])
                if not len(at):
                    continue
                with np.errstate(all="ignore"):
                    w = np.exp(s[i, at] - s[i, at].max())
                    w /= w.sum()
                    out[i, h] = w @ v[at]
                    size[i, h] = w @ np.abs(v[at])
        return out, size

    def check(self, t, requests=None):
        """Outputs against 64 bits, and rows that nobody writes.

        An output is a sum of weights times V over the sum of the weights: each
        weight is rounded to 11 bits (2^-11 of the mean of |v|, and again in the
        sum: 2^-11 of the output), the output to fp16 (2^-11 of it); scores, sums
        and exponentials in fp32 add less than 2^-14 of the mean of |v| for scores
        below 2^6, and fp16 its least step, 2^-25."""
        got = t["out"].float().cpu().numpy().reshape(self.batch, self.nodes, self.q_heads, self.dim)
        for r in range(self.batch):
            n = self.counts[r] if r < self.active else 0
            assert (got[r, max(0, n):] == 7.0).all(), f"request {r}: rows behind the tree"
            if n <= 0 or (requests is not None and r not in requests):
                continue
            want, size = self.exact(r)
            nan = np.isnan(want)
            assert (np.isnan(got[r, :n]) == nan).all(), f"request {r}: NaN"
            inf = np.isinf(want)
            assert (got[r, :n][inf] == want[inf]).all(), f"request {r}: infinities"
            fine = ~nan & ~inf
            bound = 2.0 ** -10 * np.abs(want) + (2.0 ** -11 + 2.0 ** -14) * size + 2.0 ** -24
            off = np.abs(got[r, :n][fine] - want[fine]) / bound[fine]
            assert off.max(initial=0) <= 1.0, f"request {r}: {off.max():.2f} of the bound"
