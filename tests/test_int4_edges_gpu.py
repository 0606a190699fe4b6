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


class Arena:
    """Hands out the results and workspaces of a call from one patterned buffer, a patterned gap behind each."""

    def __init__(self, monkeypatch, nbytes=256 << 20):
        self.buf, self.at, self.gaps, self.plain = torch.full((nbytes,), 0xA5, dtype=torch.uint8, device=DEV), 0, [], torch.empty
        monkeypatch.setattr(torch, "empty", self.empty)

    def empty(self, *size, dtype=None, device=None, **kw):
        if device is None or torch.device(device).type != "cuda":
            return self.plain(*size, dtype=dtype, device=device, **kw)
        size = tuple(size[0]) if len(size) == 1 and not isinstance(size[0], int) else size
        n = torch.Size(size).numel() * dtype.itemsize
        lo, self.at = self.at, -(-(self.at + n + 4096) // 512) * 512
        assert self.at <= self.buf.numel()
        self.gaps.append((lo + n, self.at))
        return self.buf[lo: lo + n].view(dtype).view(size)

    def queries(self, q):
        """q, whose `new_empty` takes from here too."""
        arena = self

        class Queries(torch.Tensor):
            def new_empty(self, size, dtype=None):
                return arena.empty(size, dtype=dtype or self.dtype, device=DEV)
        return q.as_subclass(Queries)

    def check(self):
        assert self.gaps and all(bool((self.buf[lo:hi] == 0xA5).all()) for lo, hi in self.gaps)


# the kernel that reads 4-bit pages (8 and 16 rows), then both prompt kernels over expanded pages, with and without slices of the keys
@pytest.mark.parametrize("hq,hkv,dim,bs,new,ctx,last", [(8, 2, 128, 64, [1, 2], [90, 300], 40), (64, 4, 128, 64, [1, 3], [90, 300], 9), (64, 4, 128, 64, [70, 33], [70, 200], 150),
                                                        (64, 4, 128, 64, [16, 17], [2000, 3000], 70), (16, 4, 64, 16, [300], [411], 320), (64, 4, 128, 32, [700, 650], [800, 900], 1351)])
def test_query_boundaries_past_the_last_row(hq, hkv, dim, bs, new, ctx, last, monkeypatch):
    """A sequence that claims rows behind the last one of q has its rows where its length puts them, and nothing is written behind a result or a workspace."""
    args, _, _ = case(hq, hkv, dim, bs, new, ctx, seed=7)
    T, claimed = sum(new), new[:-1] + [last - sum(new[:-1])]
    q = torch.full((last + 300, hq, dim), 3.0, dtype=torch.bfloat16, device=DEV)
    q[:T] = args[0]
    out, spread, mass, top = dense_attention(q[:last], cache_values(args[1], dim), cache_values(args[2], dim), args[3].cpu(), claimed, ctx, args[6])
    cu = cu_of(claimed)
    arena = Arena(monkeypatch)
    got = ops.gqa_attention_paged(arena.queries(q[:T]), *args[1:4], cu, *args[5:])
    arena.check()
    monkeypatch.undo()
    assert got.untyped_storage().data_ptr() == arena.buf.untyped_storage().data_ptr()
    within(got, out[:T], attention_bound(out, spread, mass, top)[:T])
    assert bool((q[T:] == 3).all())


def test_tables_whose_rows_overlap_are_refused():
    from test_int4_edges_cpu import overlapping
    overlapping(DEV)
