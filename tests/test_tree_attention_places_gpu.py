"""Tree attention, append and keep on pages far into great pools, whose offsets pass 32 bits, and
values that fp16 holds with few bits."""
import numpy as np
import pytest
import torch

from tree_helpers import Forest

pytestmark = pytest.mark.gpu


def far(f, t, pages):
    """The pools of t as the last pages of pools of `pages`."""
    first = pages - f.pages
    out = dict(t)
    for name in ("k", "v"):
        pool = torch.empty(pages * f.page_stride, dtype=torch.float16, device="cuda")
        pool[first * f.page_stride:] = t[name]
        out[name] = pool
    out["tables"] = torch.where(t["tables"] >= 0, t["tables"] + first, t["tables"])
    return out


@pytest.mark.parametrize("nodes,qh,kvh,dim", [(5, 8, 4, 128), (20, 8, 4, 128), (64, 16, 4, 64),
                                              (5, 8, 4, 64), (6, 8, 4, 96)])
def test_pages_past_32_bits(tmc, nodes, qh, kvh, dim):
    f = Forest(71, [900, 40, 2000], nodes, qh, kvh, dim, 16)
    t = far(f, f.device(), (5 << 30) // (2 * f.page_stride))  # of 5 GiB, 2.5 2^30 elements
    f.attend(tmc, t)
    f.check(t)


@pytest.mark.parametrize("nodes,qh,kvh,dim", [(5, 8, 8, 128), (20, 8, 8, 128)])
def test_pools_of_64_gib(tmc, nodes, qh, kvh, dim):
    """16-byte units do not fit 32 bits any more."""
    f = Forest(72, [300, 40], nodes, qh, kvh, dim, 16)
    if torch.cuda.mem_get_info()[0] < 150 << 30:
        pytest.skip("150 GiB of free memory are needed")
    t = far(f, f.device(), (64 << 30) // (2 * f.page_stride) + 3)
    f.attend(tmc, t)
    f.check(t)
    del t
    torch.cuda.empty_cache()


def test_append_and_keep_past_32_bits(tmc):
    """Rows appended to the last pages of great pools and moved up there."""
    batch, nodes, heads, dim, page, pages = 3, 6, 4, 128, 16, (5 << 30) // (2 * 4 * 16 * 128)
    gen = torch.Generator(device="cuda").manual_seed(73)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    qkv = torch.randn(batch, nodes, 3 * heads * dim, generator=gen, device="cuda").half()
    cosine, sine = torch.ones(64, dim // 2, device="cuda"), torch.zeros(64, dim // 2, device="cuda")
    tables = pages - 1 - torch.arange(batch * 2, dtype=torch.int32).reshape(batch, 2).cuda()
    k, v = (torch.empty(pages, heads, page, dim, dtype=torch.float16, device="cuda") for _ in "kv")
    k[-8:], v[-8:] = 5.0, 5.0
    cached, q = i32([13, 0, 20]), torch.zeros(batch, nodes, heads * dim, device="cuda").half()
    tmc.tree_rope_append(qkv, cosine, sine, cached, i32([[0] * nodes] * batch), None, tables, None, q,
                         k, v, batch, nodes, heads, heads, dim, page, 2)
    path, accepted = i32([[0, 2, 5, -1, -1, -1], [0, 1, 3, 4, -1, -1], [0, -1, -1, -1, -1, -1]]), \
        i32([3, 4, 1])
    tmc.tree_keep([k], [v], tables[None].contiguous(), cached, path, accepted, heads, page, dim)
    for r in range(batch):
        order = [n for n in path[r].tolist() if n >= 0]
        order += list(range(len(order), nodes))  # behind the path as they were appended
        for s, n in enumerate(order):
            at = int(cached[r]) + s
            where = int(tables[r, at // page]), slice(None), at % page
            row = qkv[r, n].reshape(3, heads, dim)
            assert torch.equal(k[where], row[1]) and torch.equal(v[where], row[2]), (r, s)
    assert torch.equal(q, qkv[..., :heads * dim])


@pytest.mark.parametrize("nodes,qh,kvh", [(5, 8, 4), (14, 8, 4), (30, 8, 4), (40, 8, 2), (64, 8, 2)])
@pytest.mark.parametrize("dim", [64, 128, 96])
def test_small_values(tmc, nodes, qh, kvh, dim):
    """K and V below 2^-14, the least normal number of fp16: their bits count."""
    f = Forest(74, [500, 31], nodes, qh, kvh, dim, 16)
    f.q *= np.float16(2.0 ** 10)
    for k, v in zip(f.k, f.v):
        k *= np.float16(2.0 ** -15)
        v *= np.float16(2.0 ** -16)
    t = f.device()
    f.attend(tmc, t)
    got = t["out"].float().cpu().numpy().reshape(f.batch, nodes, qh, dim)
    for r in range(f.batch):
        want, size = f.exact(r)
        # as Forest.check(), with the least step of fp16, 2^-24, rounded by half
        bound = 2.0 ** -10 * np.abs(want) + (2.0 ** -11 + 2.0 ** -14) * size + 2.0 ** -25
        assert (np.abs(got[r] - want) <= bound).all()
