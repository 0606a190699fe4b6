"""4-bit pages on the GPU: calls at the edges of what the operators allow."""
import pytest
import torch

from int4_cases import attention_bound, cache_values, dense_attention, random_cache, softmax_scale, table_of
from nanoengine_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def cu_of(new):
    return torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=DEV)


def case(hq, hkv, dim, bs, new, ctx, window=0, seed=0):
    """Arguments of a call, its result in 64 bits and how far a result may be off."""
    g = gen(seed)
    blocks = sum(-(-c // bs) for c in ctx) + 3
    table, _, _ = table_of(ctx, bs, blocks, g)
    kc, vc = (random_cache(blocks, hkv, dim, bs, g, DEV) for _ in range(2))
    q = torch.randn(sum(new), hq, dim, generator=g).to(torch.bfloat16).cuda()
    out, spread, mass, top = dense_attention(q, cache_values(kc, dim), cache_values(vc, dim), table, new, ctx, softmax_scale(dim), window)
    return [q, kc, vc, table.cuda(), cu_of(new), torch.tensor(ctx, dtype=torch.int32, device=DEV), softmax_scale(dim), window], out, attention_bound(out, spread, mass, top)


def within(got, out, bound):
    off = (got.double() - out).abs() - bound
    assert bool((off <= 0).all()), float(off.max())


# few query rows (the kernel that reads 4-bit pages) and many (expanded pages, both prompt kernels)
@pytest.mark.parametrize("hq,hkv,dim,bs,new,ctx", [(64, 4, 128, 64, [1, 2], [70, 200]), (64, 4, 128, 64, [70, 33], [70, 200]), (16, 4, 64, 16, [300], [411]),
                                                   (64, 4, 128, 32, [700, 650], [800, 900])])
def test_block_tables_of_a_larger_batch(hq, hkv, dim, bs, new, ctx):
    args, out, bound = case(hq, hkv, dim, bs, new, ctx)
    exact = ops.gqa_attention_paged(*args)
    table = args[3]
    args[3] = torch.cat([table, torch.full((5, table.shape[1]), 2 ** 30, dtype=torch.int32, device=DEV)])
    got = ops.gqa_attention_paged(*args)
    assert torch.equal(got, exact)
    within(got, out, bound)
    with pytest.raises(ValueError, match="block table"):
        ops.gqa_attention_paged(*args[:3], table[: len(ctx) - 1], *args[4:])
