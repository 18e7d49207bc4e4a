"""The tree append beyond 2^31 elements of qkv, where element indices pass 31 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BATCH, NODES, Q_HEADS, KV_HEADS, DIM, PAGE, PAGES = 1402, 256, 32, 8, 128, 16, 18
WIDTH = (Q_HEADS + 2 * KV_HEADS) * DIM


def append(tmc, qkv, cosine, sine, tables, batch, dtype):
    """(q, K pool, V pool) of the last `batch` requests."""
    q = torch.full((batch, NODES, Q_HEADS * DIM), 7.0, dtype=dtype, device="cuda")
    pools = [torch.full((3 * PAGES, KV_HEADS, PAGE, DIM), 7.0, dtype=dtype, device="cuda")
             for _ in range(2)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    tmc.tree_rope_append(qkv[-batch:], cosine, sine, i32([11] * batch),
                         i32([[i // 2 for i in range(NODES)]] * batch), None,
                         tables[-batch:].contiguous(), None, q, *pools, batch, NODES, Q_HEADS,
                         KV_HEADS, DIM, PAGE, PAGES)
    return [q] + pools


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_append_of_more_than_31_bits(tmc, dtype):
    assert 2 ** 31 < BATCH * NODES * WIDTH < 2 ** 32
    gen = torch.Generator(device="cuda").manual_seed(51)
    qkv = torch.randn(BATCH, NODES, WIDTH, generator=gen, device="cuda", dtype=dtype)
    angle = torch.rand(200, DIM // 2, generator=gen, device="cuda") * 6.0
    tables = torch.full((BATCH, PAGES), -1, dtype=torch.int32)
    tables[-3:] = torch.arange(3 * PAGES).reshape(3, PAGES)  # the others store their queries alone
    args = qkv, angle.cos(), angle.sin(), tables.cuda()
    whole = append(tmc, *args, BATCH, dtype)
    few = append(tmc, *args, 3, dtype)
    assert torch.equal(whole[0][-3:], few[0])
    assert torch.equal(whole[1], few[1]) and torch.equal(whole[2], few[2])
    assert (few[1][few[1] != 7.0].numel() > 0) and torch.isfinite(few[0]).all()
    # every query is written, also where the element index passes 2^31
    assert not (whole[0] == 7.0).all(dim=-1).any()
    middle = 2 ** 31 // (NODES * WIDTH)  # the request at that place, by itself
    alone = append(tmc, qkv[:middle + 1], *args[1:3], args[3][:middle + 1], 1, dtype)
    assert torch.equal(whole[0][middle], alone[0][0])
