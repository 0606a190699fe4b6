"""4-bit pages on the GPU: calls at the edges of what the operators allow."""
import pytest
import torch

from int4_cases import BF16_HALF_STEP, attention_bound, cache_values, dense_attention, nearest, random_cache, rope_table, rows_exact, softmax_scale, table_of
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


@pytest.mark.parametrize("T,hq,hkv,d,sections,interleaved,norm", [(1, 4, 1, 96, [16, 16, 16], True, True), (37, 8, 2, 80, [8, 20, 12], False, True),
                                                                   (130, 4, 4, 112, [24, 16, 16], True, False), (5, 8, 2, 96, [0, 48], False, True)])
def test_several_axes_at_other_head_sizes(T, hq, hkv, d, sections, interleaved, norm):
    """Head sizes that the row kernel is not built for, bf16 caches: norm and rotation are rounded one behind the other, as with one position."""
    g = gen(d)
    qkv = torch.randn(T, (hq + 2 * hkv) * d, generator=g).to(torch.bfloat16).cuda()
    qw, kw = ((1 + 0.2 * torch.randn(d, generator=g)).to(torch.bfloat16).cuda() if norm else None for _ in range(2))
    table, pos = rope_table(d, 500, DEV), torch.randint(0, 500, (len(sections), T), generator=g).cuda()
    kc, vc = (torch.full((T // 16 + 2, 16, hkv, d), 3.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    slots = torch.randperm(kc.shape[0] * 16, generator=g)[:T].cuda()
    x = qkv.view(T, -1, d).clone()
    call = lambda: ops.gqa_qkv_prepare(qkv, hq, hkv, d, qw, kw, 1e-6, False, pos, table, kc, vc, slots, sections, interleaved)       # noqa: E731
    q = call()
    # two roundings: of the normed row (either element of a pair, turned by at most 1 each) and of the result
    h = BF16_HALF_STEP * (2 if norm else 1) * (1 + 2.0 ** -7)
    for got, rows, w in ((q, x[:, :hq], qw), (kc.flatten(0, 1)[slots], x[:, hq: hq + hkv], kw)):
        want = rows_exact(rows, w, 1e-6, 0.0, pos, table, sections, interleaved)
        size = rows_exact(rows, w, 1e-6, 0.0, torch.zeros_like(pos), table, sections, interleaved)       # normed, not turned
        a, b = size.chunk(2, -1)
        pair = (a.abs() + b.abs()).repeat(1, 1, 2)
        assert bool(((got.double() - want).abs() <= h * pair + 2.0 ** -18 * pair.amax(-1, keepdim=True)).all())
    assert torch.equal(vc.flatten(0, 1)[slots], x[:, hq + hkv:])
    # equal positions on all axes are ordinary positions, to the bit
    one = pos[:1].expand(len(sections), T)
    kc2, kc3, vc2 = kc.clone(), kc.clone(), vc.clone()
    a = ops.gqa_qkv_prepare(x.view(T, -1).clone(), hq, hkv, d, qw, kw, 1e-6, False, one, table, kc2, vc2, slots, sections, interleaved)
    b = ops.gqa_qkv_prepare(x.view(T, -1).clone(), hq, hkv, d, qw, kw, 1e-6, False, pos[0], table, kc3, vc2, slots)
    assert torch.equal(a, b) and torch.equal(kc2, kc3)
    # positions past the table stay inside it, and the call can be captured
    far = pos.clone()
    far[0, 0], far[-1, -1] = 10 ** 12, -5
    qkv.copy_(x.view(T, -1))
    want = ops.gqa_qkv_prepare(x.view(T, -1).clone(), hq, hkv, d, qw, kw, 1e-6, False, far.clamp(0, 499), table, kc2, vc2, slots, sections, interleaved)
    pos.copy_(far)
    call()
    qkv.copy_(x.view(T, -1))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    qkv.copy_(x.view(T, -1))
    graph.replay()
    assert torch.equal(got, want) and torch.equal(kc.flatten(0, 1)[slots], kc2.flatten(0, 1)[slots])


def test_an_engine_with_three_axes_and_heads_of_96():
    from nanoengine_b200 import Config, LLM, SamplingParams
    from nanoengine_b200.models.config import ModelConfig
    sp, ps = SamplingParams(temperature=0.0, max_tokens=8, ignore_eos=True), [list(range(3, 60)), list(range(100, 117))]
    got = []
    for over in (dict(), dict(mrope_section=[16, 16, 16], mrope_interleaved=True)):
        mc = ModelConfig(architecture="Qwen3MoeForCausalLM", vocab_size=512, hidden_size=256, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=2, head_dim=96,
                         intermediate_size=512, n_routed_experts=0, first_k_dense_replace=0, q_lora_rank=None, rope_theta=1e6, max_position_embeddings=4096, qk_norm=True,
                         eos_token_id=None, **over)
        llm = LLM(Config(model="small", model_config=mc, dummy_weight=True, device="cuda", kvcache_block_size=64, max_num_seqs=4, num_kvcache_blocks=32, max_model_len=256, seed=0))
        got.append([o["token_ids"] for o in sorted(llm.generate(ps, sp), key=lambda o: o["seq_id"])])
    assert got[0] == got[1]                       # text: the same position on every axis


def test_positions_in_a_column_of_a_wider_tensor():
    T, d = 12, 64
    g = gen(3)
    qkv = torch.randn(T, 4 * d, generator=g).to(torch.bfloat16).cuda()
    table, wide = rope_table(d, 99, DEV), torch.randint(0, 99, (T, 3), generator=g).cuda()
    made = []
    for pos in (wide[:, 1].contiguous(), wide[:, 1:2], wide[:, 1], wide[:, 1].int()):
        kc, vc = (torch.zeros(1, 1, ops.kv4_page_bytes(d, 16), dtype=torch.uint8, device=DEV) for _ in range(2))
        made.append((ops.gqa_qkv_prepare(qkv, 2, 1, d, None, None, 1e-6, False, pos, table, kc, vc, torch.arange(T, device=DEV)), kc))
    assert all(torch.equal(q, made[0][0]) and torch.equal(kc, made[0][1]) for q, kc in made)
    three = [wide.t(), wide.t().contiguous(), torch.cat([wide, wide], 1).t()[:3], wide.t().int()]           # rows of axes with any strides
    made = []
    for pos in three:
        kc, vc = (torch.zeros(1, 1, ops.kv4_page_bytes(d, 16), dtype=torch.uint8, device=DEV) for _ in range(2))
        made.append((ops.gqa_qkv_prepare(qkv, 2, 1, d, None, None, 1e-6, False, pos, table, kc, vc, torch.arange(T, device=DEV), [8, 12, 12]), kc))
    assert all(torch.equal(q, made[0][0]) and torch.equal(kc, made[0][1]) for q, kc in made)


@pytest.mark.parametrize("sections", [None, [8, 12, 12]])
def test_norm_weights_that_bf16_does_not_hold_are_refused(sections):
    """The plain form takes them as they are (1 + 2^-9 is 1 in bf16); the kernel has no form for them."""
    T, d = 4, 64
    qkv = torch.randn(T, 4 * d, generator=gen(1)).to(torch.bfloat16).cuda()
    pos, table = torch.zeros(3 if sections else 1, T, dtype=torch.long, device=DEV), rope_table(d, 9, DEV)
    kc = torch.zeros(1, 1, ops.kv4_page_bytes(d, 16), dtype=torch.uint8, device=DEV)
    good, odd = torch.ones(d, dtype=torch.bfloat16, device=DEV), torch.ones(d, device=DEV) + 2.0 ** -9
    for qw, kw in ((odd, good), (good, odd), (good[:32], good)):
        with pytest.raises(ValueError, match="norm weights"):
            ops.gqa_qkv_prepare(qkv, 2, 1, d, qw, kw, 1e-6, False, pos if sections else pos[0], table, kc, kc.clone(), torch.arange(T, device=DEV), sections)
    assert not kc.any()


@pytest.mark.parametrize("d,T", [(64, 40000), (128, 40000), (256, 20000)])
def test_codes_of_many_key_rows_are_those_of_64_bits(d, T):
    """Ten million elements a size: some lie nearer to a border than the 32-bit error allows to tell."""
    g = torch.Generator(device=DEV).manual_seed(d)
    hkv, bs = 4, 64
    qkv = torch.randn(T, 3 * hkv * d, generator=g, device=DEV).to(torch.bfloat16)
    kw = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(torch.bfloat16)
    pos, table = torch.randint(0, 4000, (3, T), generator=g, device=DEV), rope_table(d, 4000, DEV)
    kc, vc = (torch.zeros(-(-T // bs), hkv, ops.kv4_page_bytes(d, bs), dtype=torch.uint8, device=DEV) for _ in range(2))
    sec = [d // 4, d // 8, d // 8]
    ops.gqa_qkv_prepare(qkv, hkv, hkv, d, kw, kw, 1e-6, True, pos, table, kc, vc, torch.arange(T, device=DEV), sec, True)
    want = nearest(rows_exact(qkv.view(T, -1, d)[:, hkv: 2 * hkv], kw, 1e-6, 1.0, pos, table, sec, True))
    assert torch.equal(cache_values(kc, d).flatten(0, 1)[:T], want)


@pytest.mark.parametrize("kv", ["int4", "auto"])
def test_the_room_of_expanded_pages_stays_outside_the_cache(kv, monkeypatch):
    """A cache sized from free memory leaves what the widest prompt step over it expands."""
    from nanoengine_b200 import Config, LLM, SamplingParams
    from nanoengine_b200.models.config import ModelConfig
    from nanoengine_b200.ops import sm100_attn
    from nanoengine_b200.runtime import model_runner
    seen, plain = [], model_runner.kv_budget_blocks

    def budget(*a, reserved=0, **kw):
        seen.append(reserved)
        return min(300, plain(*a, reserved=reserved, **kw))

    monkeypatch.setattr(model_runner, "kv_budget_blocks", budget)
    mc = ModelConfig(architecture="Qwen3MoeForCausalLM", vocab_size=512, hidden_size=256, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=2, head_dim=128,
                     intermediate_size=512, n_routed_experts=0, first_k_dense_replace=0, q_lora_rank=None, rope_theta=1e6, max_position_embeddings=8192, qk_norm=True,
                     eos_token_id=None)
    llm = LLM(Config(model="small", model_config=mc, dummy_weight=True, device="cuda", kv_cache_dtype=kv, kvcache_block_size=64, max_num_seqs=4, max_num_batched_tokens=1024,
                     max_model_len=4096, gpu_memory_utilization=0.2, enforce_eager=True, seed=0))
    assert seen == [sm100_attn.int4_expansion_room(1024, 4, 4096, 8, 2, 128, 64) if kv == "int4" else 0]
    # a portion of 1000 tokens behind 3000: no more than that is taken beside the cache
    sp = SamplingParams(temperature=0.0, max_tokens=1, ignore_eos=True)
    llm.generate([[5 + i % 400 for i in range(3900)]], sp)
    assert kv == "auto" or seen[0] >= 4 * 3904 * 2 * 128


KEPT = [
    # hq, hkv, dim, block size, new, contexts, window: row tiles of 8 and of 16, tiles that lie in a page and that do not, contexts cut into pieces and not
    (16, 2, 256, 64, [1] * 5, [300, 1, 64, 65, 2000], 0),
    (16, 2, 256, 16, [4, 3], [90, 700], 0),
    (64, 4, 256, 64, [1, 2], [40, 5000], 0),
    (16, 4, 64, 64, [1, 1], [129, 3000], 0),
    (32, 2, 64, 32, [1, 3], [77, 1500], 0),
    (32, 8, 128, 64, [1, 1], [900, 64], 100),
    (64, 4, 128, 16, [1, 2], [900, 333], 70),
    (16, 2, 256, 64, [2], [3001], 1000),
]


@pytest.mark.parametrize("hq,hkv,dim,bs,new,ctx,window", KEPT)
def test_probabilities_of_windows_and_of_heads_that_are_not_128_wide_keep_17_bits(hq, hkv, dim, bs, new, ctx, window):
    """As over bf16 pages.  Weights w_i (1 + d_i), |d_i| <= e = 2^-17 (a probability as bf16, off by at most 2^-8 of its power of two, and the rest as bf16 again, normalised by
    their own sum, are off by e (1 + 2 e) sum w |v - o|; the result is rounded once; 32-bit scores and exponentials as in `attention_bound`."""
    from nanoengine_b200.ops import sm100_attn
    args, out, _ = case(hq, hkv, dim, bs, new, ctx, window, seed=12)
    _, spread, mass, top = dense_attention(args[0], cache_values(args[1], dim), cache_values(args[2], dim), args[3].cpu(), new, ctx, args[6], window)
    e = 2.0 ** -17
    before = sm100_attn.INT4_CALLS[0]
    got = ops.gqa_attention_paged(*args)
    assert sm100_attn.INT4_CALLS[0] == before + 1
    within(got, out, BF16_HALF_STEP * out.abs() + (1 + BF16_HALF_STEP) * (e * (1 + 2 * e) * spread + (2.0 ** -15 * top + 2.0 ** -18) * mass) + 1e-30)
