"""4-bit key / value rows, positions on several axes and the step tables on the GPU against 64-bit statements."""
import pytest
import torch

from int4_cases import BF16_HALF_STEP, attention_bound, cache_values, dense_attention, nearest, random_cache, rope_table, rows_exact, softmax_scale, table_of, tables_exact
from nanoengine_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def cu_of(new):
    return torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=DEV)


# ---- tables -----------------------------------------------------------------------------------------------------------------------
TABLES = [
    # block size, new, ctx, rows, padding, tokens beyond, columns beyond
    (64, [1, 1, 1], [1, 64, 65], 3, 1, 0, 0),
    (64, [1] * 128, [63 + 17 * i for i in range(128)], 144, 1, 0, 3),
    (16, [5, 0, 20], [5, 9, 33], 4, 3, 6, 0),
    (1, [2, 3], [7, 3], 2, 1, 0, 1),
    (64, [3000, 1, 777], [3000, 900, 1000], 3, 1, 5, 0),
    (64, [1], [131072], 1, 1, 0, 0),
    (16, [1] * 700, [1 + i % 50 for i in range(700)], 701, 2, 0, 0),
    (32, [], [], 2, 2, 1, 1),
    (32, [], [], 0, 1, 3, 0),
]


@pytest.mark.parametrize("bs,new,ctx,rows,pad,extra,wide", TABLES)
def test_step_tables(bs, new, ctx, rows, pad, extra, wide):
    table, ids, off = table_of(ctx, bs, 40000 if bs > 1 else 40, gen(1))
    width, tokens = table.shape[1] + wide, sum(new) + (rows - len(new)) * pad + extra
    dev = [torch.tensor(t, dtype=torch.int32, device=DEV) for t in (new, ctx)] + [ids.cuda(), off.cuda()]
    got = ops.step_tables(*dev, bs, tokens, width, rows, pad, 50000)
    want = tables_exact(new, ctx, ids.tolist(), off.tolist(), bs, tokens, width, rows, pad, 50000)
    for name, a, b in zip(got._fields, got, want):
        assert a.dtype == b.dtype and torch.equal(a.cpu(), b), name


def test_step_tables_of_bad_lengths_and_pages_store_nothing():
    new, ctx, bs = [3, 2, 4, -2], [1, 40, 100, 5], 16
    ids, off = torch.tensor([4, -7, 2, 9], dtype=torch.int32), torch.tensor([0, 1, 3, 9, -4], dtype=torch.int32)
    got = ops.step_tables(torch.tensor(new, device=DEV), torch.tensor(ctx, device=DEV), ids.cuda(), off.cuda(), bs, 11, 3)
    want = tables_exact(new, ctx, ids.tolist(), off.tolist(), bs, 11, 3, 4, 1, -1)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


def test_step_tables_write_the_front_of_larger_buffers_and_replay():
    bs, width, rows, tokens = 64, 5, 6, 9
    big = ops.StepTables(*(torch.full(s, -5, dtype=t, device=DEV) for s, t in (((9,), torch.int32), ((8,), torch.int32), ((11,), torch.int64), ((11,), torch.int64),
                                                                                ((8, 7), torch.int32), ((8,), torch.int32))))
    new, ctx, off = (torch.zeros(n, dtype=torch.int32, device=DEV) for n in (4, 4, 5))
    ids = torch.zeros(20, dtype=torch.int32, device=DEV)
    call = lambda: ops.step_tables(new, ctx, ids, off, bs, tokens, width, rows, 1, 77, out=big)         # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for n, c in (([1, 1, 1, 1], [5, 64, 65, 300]), ([2, 1, 3, 1], [2, 129, 200, 64])):
        table, i, o = table_of(c, bs, 20, gen(sum(c)))
        new.copy_(torch.tensor(n)), ctx.copy_(torch.tensor(c)), off.copy_(o), ids[: i.numel()].copy_(i)
        for t in big:
            t.fill_(-5)
        graph.replay()
        want = tables_exact(n, c, ids.tolist(), o.tolist(), bs, tokens, width, rows, 1, 77)
        for a, b, whole in zip(got, want, big):
            assert torch.equal(a.cpu(), b)
            left = whole.clone()
            left[tuple(slice(k) for k in b.shape)] = -5
            assert bool((left == -5).all())


# ---- rows -------------------------------------------------------------------------------------------------------------------------
def rows_inputs(T, hq, hkv, d, axes, seed, top=500):
    g = gen(seed)
    qkv = torch.randn(T, (hq + 2 * hkv) * d, generator=g).to(torch.bfloat16).cuda()
    qw, kw = ((torch.rand(d, generator=g) + 0.5).to(torch.bfloat16).cuda() for _ in range(2))
    pos = torch.randint(0, top, (axes, T), generator=g).cuda()
    return g, qkv, qw, kw, pos, rope_table(d, top, DEV)


ROWS = [
    # tokens, hq, hkv, dim, block size, sections (None: one position), interleaved, norm, unit offset
    (1, 4, 1, 128, 64, None, False, True, False),
    (37, 8, 2, 128, 64, [16, 24, 24], False, True, False),
    (64, 64, 4, 128, 64, [24, 20, 20], True, True, True),
    (129, 16, 2, 256, 64, [40, 44, 44], True, True, True),
    (50, 4, 4, 64, 16, [32], False, False, False),
    (33, 3, 1, 32, 8, [4, 4, 4, 4], False, True, False),
    (20, 5, 5, 64, 128, [0, 20, 12], False, False, False),
    (300, 24, 2, 128, 32, None, False, True, False),
]


@pytest.mark.parametrize("T,hq,hkv,d,bs,sections,interleaved,norm,offset", ROWS)
@pytest.mark.parametrize("int4", [True, False])
def test_rows(T, hq, hkv, d, bs, sections, interleaved, norm, offset, int4):
    if not int4 and sections is None:
        pytest.skip("one position and bf16 rows: the ordinary front end")
    axes = 1 if sections is None else len(sections)
    g, qkv, qw, kw, pos, table = rows_inputs(T, hq, hkv, d, axes, T)
    if not norm:
        qw = kw = None
    blocks = T // bs + 3
    # the rows in front of the cache: a slot of -1 must not reach them
    if int4:
        kc, vc = (torch.full((blocks, hkv, ops.kv4_page_bytes(d, bs)), 0x5A, dtype=torch.uint8, device=DEV) for _ in range(2))
    else:
        kc, vc = (torch.full((blocks, bs, hkv, d), 3.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    slots = torch.randperm(blocks * bs, generator=g)[:T].cuda()
    if T > 4:
        slots[1] = -1
        if int4:
            slots[2] = blocks * bs                         # behind the cache: not stored
    before = [c.clone() for c in (kc, vc)]
    q = ops.gqa_qkv_prepare(qkv, hq, hkv, d, qw, kw, 1e-6, offset, pos[0] if sections is None else pos, table, kc, vc, slots, sections, interleaved)
    sec = [d // 2] if sections is None else sections
    x = qkv.view(T, -1, d)
    want_q = rows_exact(x[:, :hq], qw, 1e-6, float(offset), pos, table, sec, interleaved)
    want_k = rows_exact(x[:, hq: hq + hkv], kw, 1e-6, float(offset), pos, table, sec, interleaved)
    # one rounding of a 32-bit result: half a step, and 2^-20 of the row for the sums of two products behind a norm
    near = lambda a, b: bool(((a.double() - b).abs() <= BF16_HALF_STEP * b.abs() + 2.0 ** -20 * b.abs().amax(-1, keepdim=True)).all())      # noqa: E731
    assert near(q, want_q)
    live = (slots >= 0) & (slots < blocks * bs)
    at = slots[live]
    for cache, was, want in ((kc, before[0], want_k), (vc, before[1], x[:, hq + hkv:].double())):
        if int4:
            rows, old = cache_values(cache, d).flatten(0, 1), cache_values(was, d).flatten(0, 1)
            assert torch.equal(rows[at], nearest(want[live]))
        else:
            rows, old = cache.flatten(0, 1), was.flatten(0, 1)
            assert near(rows[at], want[live])
        same = torch.ones(blocks * bs, dtype=torch.bool, device=DEV)
        same[at] = False
        assert torch.equal(rows[same], old[same])
    if int4:
        k, v = ops.gqa_kv_gather(kc, vc, slots, d)
        assert torch.equal(k.double(), torch.where(live[:, None, None], cache_values(kc, d).flatten(0, 1)[slots.clamp(0, blocks * bs - 1)], 0.0))
        assert torch.equal(v.double(), torch.where(live[:, None, None], cache_values(vc, d).flatten(0, 1)[slots.clamp(0, blocks * bs - 1)], 0.0))


@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("eps", [1e-6, 0.0])
def test_key_rows_whose_squares_32_bits_do_not_hold(d, eps):
    """Keys of 2^-70 to 2^100 (a row of ordinary size among them): the codes are those of the row in 64 bits all the same."""
    T, hq, hkv, bs = 9, 2, 3, 16
    g, qkv, qw, kw, pos, table = rows_inputs(T, hq, hkv, d, 1, d)
    size = torch.tensor([-70, -64, -40, -1, 0, 30, 63, 64, 100], device=DEV)
    qkv = (qkv.float() * torch.exp2(size.float())[:, None]).to(torch.bfloat16)
    kc, vc = (torch.zeros(2, hkv, ops.kv4_page_bytes(d, bs), dtype=torch.uint8, device=DEV) for _ in range(2))
    ops.gqa_qkv_prepare(qkv, hq, hkv, d, qw, kw, eps, False, pos[0], table, kc, vc, torch.arange(T, device=DEV))
    x = qkv.view(T, -1, d)
    for cache, want in ((kc, rows_exact(x[:, hq: hq + hkv], kw, eps, 0.0, pos, table, [d // 2], False)), (vc, x[:, hq + hkv:].double())):
        most = 7 * 1.875 * 2.0 ** 15
        assert torch.equal(cache_values(cache, d).flatten(0, 1)[:T], nearest(want.clamp(-most, most)))


@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_store_alone_takes_strided_rows_and_extremes(d):
    g = gen(d)
    T, hkv, bs = 21, 3, 16
    wide = (torch.randn(T, 2 * hkv * d + 5, generator=g) * torch.exp2(torch.randint(-20, 20, (T, 1), generator=g).float())).to(torch.bfloat16).cuda()
    k, v = wide[:, : hkv * d].view(T, hkv, d), wide[:, hkv * d + 1: 2 * hkv * d + 1].unflatten(1, (hkv, d))       # the values start at an odd element
    k[0, 0, :3] = torch.tensor([float("inf"), -float("inf"), float("nan")])
    v[3] = float("nan")
    v[4] = 0
    kc, vc = (torch.zeros(4, hkv, ops.kv4_page_bytes(d, bs), dtype=torch.uint8, device=DEV) for _ in range(2))
    slots = torch.randperm(4 * bs, generator=g)[:T].cuda()
    ops.gqa_kv_store(kc, vc, slots, k, v)
    from nanoengine_b200.ops import reference as ref
    for cache, x in ((kc, k), (vc, v)):
        want = ref.kv4_values(*ref.kv4_quant(x.cpu())).double()
        assert torch.equal(cache_values(cache, d).flatten(0, 1)[slots].cpu(), want)


def test_positions_past_the_table_stay_inside_it():
    g, qkv, qw, kw, pos, table = rows_inputs(6, 2, 1, 64, 3, 4, top=50)
    kc, vc = (torch.zeros(1, 1, ops.kv4_page_bytes(64, 16), dtype=torch.uint8, device=DEV) for _ in range(2))
    bad = pos.clone()
    bad[0, 1], bad[2, 3] = 10 ** 12, -7
    a = ops.gqa_qkv_prepare(qkv, 2, 1, 64, qw, kw, 1e-6, False, bad, table, kc, vc, torch.arange(6, device=DEV), [12, 10, 10])
    b = ops.gqa_qkv_prepare(qkv, 2, 1, 64, qw, kw, 1e-6, False, bad.clamp(0, 49), table, kc, vc, torch.arange(6, device=DEV), [12, 10, 10])
    assert torch.equal(a, b)


def test_equal_positions_on_all_axes_are_ordinary_positions():
    T, d = 40, 128
    g, qkv, qw, kw, pos, table = rows_inputs(T, 8, 2, d, 1, 2)
    made = []
    for p, sec in ((pos[0], None), (pos.expand(3, T), [24, 20, 20])):
        kc, vc = (torch.zeros(2, 2, ops.kv4_page_bytes(d, 64), dtype=torch.uint8, device=DEV) for _ in range(2))
        made.append((ops.gqa_qkv_prepare(qkv, 8, 2, d, qw, kw, 1e-6, False, p, table, kc, vc, torch.arange(T, device=DEV), sec, True), kc, vc))
    assert all(torch.equal(a, b) for a, b in zip(*made))


def test_rows_of_a_strided_projection():
    T, hq, hkv, d = 30, 4, 2, 128
    g, qkv, qw, kw, pos, table = rows_inputs(T, hq, hkv, d, 3, 8)
    wide = torch.zeros(T, qkv.shape[1] + 9, dtype=torch.bfloat16, device=DEV)
    for first in (0, 1, 8):
        wide[:, first: first + qkv.shape[1]] = qkv
        made = []
        for x in (qkv, wide[:, first: first + qkv.shape[1]]):
            kc, vc = (torch.zeros(2, hkv, ops.kv4_page_bytes(d, 16), dtype=torch.uint8, device=DEV) for _ in range(2))
            made.append((ops.gqa_qkv_prepare(x, hq, hkv, d, qw, kw, 1e-6, False, pos.t().contiguous().t(), table, kc, vc, torch.arange(T, device=DEV), [16, 24, 24]), kc, vc))
        assert all(torch.equal(a, b) for a, b in zip(*made))


def test_a_rotary_table_at_an_odd_place():
    g, qkv, qw, kw, pos, table = rows_inputs(7, 8, 2, 128, 1, 3)
    wide = torch.zeros(table.numel() + 3, device=DEV)
    made = []
    for first in (None, 1, 3):
        if first is not None:
            wide[first: first + table.numel()] = table.flatten()
        t = table if first is None else wide[first: first + table.numel()].view_as(table)
        kc, vc = (torch.zeros(2, 2, ops.kv4_page_bytes(128, 16), dtype=torch.uint8, device=DEV) for _ in range(2))
        made.append((ops.gqa_qkv_prepare(qkv, 8, 2, 128, qw, kw, 1e-6, False, pos[0], t, kc, vc, torch.arange(7, device=DEV)), kc, vc))
    for other in made[1:]:
        assert all(torch.equal(a, b) for a, b in zip(made[0], other))


@pytest.mark.parametrize("d,bs", [(32, 4), (32, 12), (64, 2), (64, 6), (128, 1), (128, 3), (256, 1), (256, 5)])
def test_small_and_odd_pages_of_whole_words(d, bs):
    T, hkv = 11, 3
    blocks = T // bs + 2
    k, v = (torch.randn(T, hkv, d, generator=gen(d + bs)).to(torch.bfloat16).cuda() for _ in range(2))
    kc, vc = (torch.zeros(blocks, hkv, ops.kv4_page_bytes(d, bs), dtype=torch.uint8, device=DEV) for _ in range(2))
    slots = torch.randperm(blocks * bs, generator=gen(1))[:T].cuda()
    ops.gqa_kv_store(kc, vc, slots, k, v)
    for cache, want, got in zip((kc, vc), (k, v), ops.gqa_kv_gather(kc, vc, slots, d)):
        assert torch.equal(cache_values(cache, d).flatten(0, 1)[slots], nearest(want)) and torch.equal(got.double(), nearest(want))


# ---- attention --------------------------------------------------------------------------------------------------------------------
ATTENTION = [
    # hq, hkv, dim, block size, new tokens, contexts, window
    (4, 1, 128, 64, [1], [1], 0),
    (64, 4, 128, 64, [1, 1, 1, 1], [1, 64, 65, 700], 0),
    (16, 2, 256, 64, [1, 1, 1], [63, 129, 1000], 0),
    (16, 4, 64, 64, [1, 1], [300, 5], 0),
    (8, 8, 128, 64, [1, 3, 0, 2], [90, 65, 7, 2], 0),
    (24, 2, 128, 64, [1, 2], [200, 130], 0),
    (20, 1, 64, 64, [1, 1], [77, 1], 0),                               # a group of more than 16 heads
    (40, 1, 128, 64, [2], [500], 0),
    (3, 1, 64, 64, [4, 1], [4, 260], 0),
    (10, 2, 128, 64, [3, 1], [66, 128], 0),
    (32, 8, 128, 16, [4, 4, 1], [100, 17, 16], 0),
    (8, 2, 256, 32, [2], [333], 0),
    (8, 2, 64, 128, [1, 2], [129, 640], 0),
    (64, 4, 128, 64, [1, 1, 2], [900, 64, 65], 100),
    (8, 1, 128, 64, [5], [200], 3),
    (8, 1, 128, 16, [1], [50], 1),
    (12, 4, 128, 64, [5], [3], 0),                                     # more new tokens than context: the first see nothing
    (8, 2, 128, 64, [1, 1, 0], [0, 40, 0], 0),
    (32, 8, 128, 64, [1], [5000], 0),                                  # sliced keys
    (8, 1, 128, 64, [1, 1], [9000, 70], 0),
    (16, 2, 256, 64, [1], [7000], 3000),
]


def run_attention(hq, hkv, dim, bs, new, ctx, window, seed=0, q=None):
    g = gen(seed)
    blocks = sum(-(-c // bs) for c in ctx) + 3
    table, _, _ = table_of(ctx, bs, blocks, g)
    kc, vc = (random_cache(blocks, hkv, dim, bs, g, DEV) for _ in range(2))
    q = torch.randn(sum(new), hq, dim, generator=g).to(torch.bfloat16).cuda() if q is None else q
    args = (q, kc, vc, table.cuda(), cu_of(new), torch.tensor(ctx, dtype=torch.int32, device=DEV), softmax_scale(dim), window)
    return args, dense_attention(q, cache_values(kc, dim), cache_values(vc, dim), table, new, ctx, softmax_scale(dim), window)


@pytest.mark.parametrize("hq,hkv,dim,bs,new,ctx,window", ATTENTION)
def test_attention(hq, hkv, dim, bs, new, ctx, window):
    args, (out, spread, mass, top) = run_attention(hq, hkv, dim, bs, new, ctx, window)
    got = ops.gqa_attention_paged(*args)
    off = (got.double() - out).abs() - attention_bound(out, spread, mass, top)
    assert bool((off <= 0).all()), float(off.max())


PROMPTS = [
    (64, 4, 128, 64, [70, 33], [70, 200], 0),
    (16, 2, 256, 64, [65], [90], 0),
    (16, 4, 64, 16, [40, 100], [55, 100], 0),
    (8, 8, 128, 32, [130], [131], 0),
    (32, 8, 128, 128, [64, 20], [64, 300], 25),
    (24, 2, 128, 64, [50], [80], 0),
    (9, 3, 64, 64, [90], [95], 0),                                     # three heads a group: no prompt kernel, the 4-bit one
]


@pytest.mark.parametrize("hq,hkv,dim,bs,new,ctx,window", PROMPTS)
def test_prompts(hq, hkv, dim, bs, new, ctx, window):
    args, (out, spread, mass, top) = run_attention(hq, hkv, dim, bs, new, ctx, window, seed=1)
    got = ops.gqa_attention_paged(*args)
    off = (got.double() - out).abs() - attention_bound(out, spread, mass, top)
    assert bool((off <= 0).all()), float(off.max())


# at most eight rows of a kv head per sequence: the products with keys and dims as their rows
FEW_ROWS = [
    # hq, hkv, dim, block size, new tokens, contexts, window
    (8, 8, 128, 64, [1, 1, 1], [1, 64, 193], 0),
    (4, 2, 128, 16, [1, 1], [17, 300], 0),
    (6, 2, 64, 32, [1, 1], [95, 96], 0),
    (10, 2, 256, 64, [1], [1025], 0),
    (6, 1, 128, 192, [1, 1], [700, 191], 0),
    (14, 2, 64, 64, [1, 1], [2000, 3], 0),
    (8, 1, 256, 16, [1, 1], [33, 31], 0),
    (32, 4, 128, 64, [1, 1], [900, 64], 100),
    (8, 2, 64, 16, [1], [77], 1),
    (16, 8, 256, 128, [4], [260], 130),
    (4, 2, 128, 64, [4, 1, 0, 3], [4, 130, 9, 2], 0),                  # more new tokens than context: the first see nothing
    (4, 1, 128, 64, [1, 0, 1], [0, 0, 5000], 0),
    (12, 1, 64, 64, [1, 0], [400, 5], 0),                              # fewer tokens than sequences: two tiles of the group's heads
    (32, 8, 128, 64, [1], [40000], 0),
    (16, 2, 256, 64, [1] * 9, [3000 + 7 * i for i in range(9)], 0),
]


@pytest.mark.parametrize("hq,hkv,dim,bs,new,ctx,window", FEW_ROWS)
def test_few_rows(hq, hkv, dim, bs, new, ctx, window):
    assert sum(new) * (hq // hkv) <= 8 * len(new)
    args, (out, spread, mass, top) = run_attention(hq, hkv, dim, bs, new, ctx, window, seed=2)
    got = ops.gqa_attention_paged(*args)
    off = (got.double() - out).abs() - attention_bound(out, spread, mass, top)
    assert bool((off <= 0).all()), float(off.max())


@pytest.mark.parametrize("hq,hkv,dim,bs,new,ctx,window", [(64, 4, 128, 64, [70, 33], [70, 200], 0), (16, 4, 64, 16, [300], [411], 0)])
def test_prompts_with_and_without_room_for_bf16_pages(hq, hkv, dim, bs, new, ctx, window, monkeypatch):
    from nanoengine_b200.ops import sm100_attn
    args, (out, spread, mass, top) = run_attention(hq, hkv, dim, bs, new, ctx, window, seed=3)
    bound = attention_bound(out, spread, mass, top)
    for room in (sm100_attn._INT4_EXPANDED_BYTES, 0):
        monkeypatch.setattr(sm100_attn, "_INT4_EXPANDED_BYTES", room)
        before = sm100_attn.INT4_CALLS[0]
        got = ops.gqa_attention_paged(*args)
        assert (sm100_attn.INT4_CALLS[0] == before) == (room > 0)
        assert bool(((got.double() - out).abs() <= bound).all())


def test_a_query_that_is_no_number_among_few_rows_stays_its_own():
    args, (out, spread, mass, top) = run_attention(16, 4, 128, 64, [1, 1], [90, 300], 0, seed=6)
    q = args[0].clone()
    q[0, 3], q[1, 5] = float("nan"), float("inf")
    got = ops.gqa_attention_paged(q, *args[1:])
    hurt = torch.zeros(got.shape[:2], dtype=torch.bool, device=DEV)
    hurt[0, 3] = hurt[1, 5] = True
    assert bool(got[hurt].isnan().all())
    assert bool(((got.double() - out).abs() <= attention_bound(out, spread, mass, top))[~hurt].all())


def test_boundaries_past_the_last_query_row_write_nothing_behind_it():
    """Query boundaries that name more rows than there are: the rows there are get their results, the kernel stays inside its tables."""
    args, (out, spread, mass, top) = run_attention(8, 2, 128, 64, [1, 2], [90, 300], 0, seed=7)
    q, kc, vc, table, _, ctx, scale, _ = args
    got = ops.gqa_attention_paged(q, kc, vc, table, torch.tensor([0, 1, 40], dtype=torch.int32, device=DEV), ctx, scale)
    assert bool(((got[:1].double() - out[:1]).abs() <= attention_bound(out, spread, mass, top)[:1]).all())
    assert got.shape == q.shape


@pytest.mark.parametrize("new", [[1, 1], [80, 90]])
def test_pages_outside_the_cache_read_as_zeros_and_contexts_end_with_their_tables(new):
    g = gen(8)
    for bs in (16, 64):
        kc, vc = (random_cache(5, 2, 128, bs, g, DEV) for _ in range(2))
        table = torch.tensor([[2, -1, 4, 70000], [5, 1, 0, 3]], dtype=torch.int32)
        ctx = [3 * bs + 5, 1000]
        n = [min(new[0], ctx[0]), min(new[1], 4 * bs)]
        q = torch.randn(sum(n), 8, 128, generator=g).to(torch.bfloat16).cuda()
        got = ops.gqa_attention_paged(q, kc, vc, table.cuda(), cu_of(n), torch.tensor(ctx, dtype=torch.int32, device=DEV), 0.08)
        out, spread, mass, top = dense_attention(q, cache_values(kc, 128), cache_values(vc, 128), table, n, ctx, 0.08)
        assert bool(((got.double() - out).abs() <= attention_bound(out, spread, mass, top)).all())


def test_strided_queries_another_stream_and_a_replayed_graph():
    args, (out, spread, mass, top) = run_attention(32, 8, 128, 64, [1, 1, 1], [130, 1000, 64], 0, seed=4)
    bound = attention_bound(out, spread, mass, top)
    q = args[0]
    wide = torch.zeros(3, 32 * 128 + 3, dtype=torch.bfloat16, device=DEV)
    for first in (0, 3):
        wide[:, first: first + 4096] = q.view(3, -1)
        got = ops.gqa_attention_paged(wide[:, first: first + 4096].unflatten(1, (32, 128)), *args[1:])
        assert bool(((got.double() - out).abs() <= bound).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.gqa_attention_paged(*args)
    side.synchronize()
    assert torch.equal(other, got)
    graphs = []
    for _ in range(2):                                                 # two captures of one call, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = ops.gqa_attention_paged(*args)
        graphs.append((graph, r))
    for graph, r in graphs + graphs:
        r.fill_(7.0)
        graph.replay()
        assert torch.equal(r, got)


def test_queries_that_are_no_numbers_stay_their_own():
    args, (out, spread, mass, top) = run_attention(16, 2, 128, 64, [2, 1], [90, 300], 0, seed=5)
    q = args[0].clone()
    q[0, 3] = float("nan")
    got = ops.gqa_attention_paged(q, *args[1:])
    hurt = torch.zeros(got.shape[:2], dtype=torch.bool, device=DEV)
    hurt[0, 3] = True
    assert bool(got[hurt].isnan().all())
    assert bool(((got.double() - out).abs() <= attention_bound(out, spread, mass, top))[~hurt].all())


def test_a_page_past_two_gigabytes():
    """Pages whose bytes lie past 2^31 of a cache: 64-bit addresses in the store, the gather and the attention."""
    blocks = (1 << 31) // ops.kv4_page_bytes(128, 64) + 8
    kc, vc = (torch.zeros(blocks, 1, ops.kv4_page_bytes(128, 64), dtype=torch.uint8, device=DEV) for _ in range(2))
    k, v = (torch.randn(64, 1, 128, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    slots = (blocks - 1) * 64 + torch.arange(64, device=DEV)
    ops.gqa_kv_store(kc, vc, slots, k, v)
    a, b = ops.gqa_kv_gather(kc, vc, slots, 128)
    assert torch.equal(a.double(), nearest(k)) and torch.equal(b.double(), nearest(v))
    assert int(kc[: blocks - 1].max()) == 0 and int(vc[: blocks - 1].max()) == 0
    q = torch.randn(1, 8, 128, device=DEV, dtype=torch.bfloat16)
    table = torch.tensor([[blocks - 1]], dtype=torch.int32)
    got = ops.gqa_attention_paged(q, kc, vc, table.cuda(), cu_of([1]), torch.tensor([64], dtype=torch.int32, device=DEV), 0.09)
    out, spread, mass, top = dense_attention(q, cache_values(kc[-1:], 128), cache_values(vc[-1:], 128), torch.zeros(1, 1, dtype=torch.int32), [1], [64], 0.09)
    assert bool(((got.double() - out).abs() <= attention_bound(out, spread, mass, top)).all())


# ---- together ---------------------------------------------------------------------------------------------------------------------
def test_a_prompt_and_decode_steps_through_all_of_them():
    """Tables, rows and attention as a model's layer runs them: a prompt, then single tokens, against 64 bits over the rows as the format holds them."""
    hq, hkv, d, bs, steps = 8, 2, 128, 64, 3
    lens = [70, 5, 130]
    g = gen(11)
    total = [n + steps for n in lens]
    table, ids, off = table_of(total, bs, 12, g)
    kc, vc = (torch.zeros(13, hkv, ops.kv4_page_bytes(d, bs), dtype=torch.uint8, device=DEV) for _ in range(2))
    rope, sec = rope_table(d, 400, DEV), [24, 20, 20]
    qw, kw = ((torch.rand(d, generator=g) + 0.5).to(torch.bfloat16).cuda() for _ in range(2))
    seen = [[] for _ in lens]                                          # 64-bit keys and values of every sequence so far
    for step in range(steps + 1):
        new = lens if step == 0 else [1] * 3
        ctx = [n + step for n in lens]
        st = ops.step_tables(torch.tensor(new, device=DEV), torch.tensor(ctx, device=DEV), ids.cuda(), off.cuda(), bs, sum(new) + 1, table.shape[1], 4, 1, 12)
        T = sum(new) + 1                                               # one padding row on the scratch page
        qkv = torch.randn(T, (hq + 2 * hkv) * d, generator=g).to(torch.bfloat16).cuda()
        pos = torch.stack([st.positions, st.positions // 3, st.positions % 7])
        q = ops.gqa_qkv_prepare(qkv, hq, hkv, d, qw, kw, 1e-6, False, pos, rope, kc, vc, st.slot_mapping, sec, True)
        got = ops.gqa_attention_paged(q, kc, vc, st.block_tables, st.cu_seqlens_q, st.context_lens, softmax_scale(d))
        x = qkv.view(T, -1, d)
        k = nearest(rows_exact(x[:, hq: hq + hkv], kw, 1e-6, 0.0, pos, rope, sec, True))
        v = nearest(x[:, hq + hkv:])
        at = 0
        for i, n in enumerate(new):
            seen[i].append((k[at: at + n], v[at: at + n]))
            kk, vv = (torch.cat(parts) for parts in zip(*seen[i]))
            one = torch.zeros(1, 1, dtype=torch.int32)
            out, spread, mass, top = dense_attention(q[at: at + n], kk[None], vv[None], one, [n], [ctx[i]], softmax_scale(d))
            assert bool(((got[at: at + n].double() - out).abs() <= attention_bound(out, spread, mass, top)).all()), (step, i)
            at += n


# ---- refusals ---------------------------------------------------------------------------------------------------------------------
def test_refusals():
    kc = torch.zeros(2, 1, ops.kv4_page_bytes(64, 16), dtype=torch.uint8, device=DEV)
    q, cu, ctx, bt = torch.zeros(1, 2, 64, device=DEV, dtype=torch.bfloat16), cu_of([1]), torch.ones(1, dtype=torch.int32, device=DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    odd = torch.zeros(2, 1, ops.kv4_page_bytes(64, 24), dtype=torch.uint8, device=DEV)
    small = torch.zeros(2, 1, ops.kv4_page_bytes(32, 16), dtype=torch.uint8, device=DEV)
    for args in ((q, kc[:, :, :-1], kc[:, :, :-1], bt, cu, ctx, 0.1), (q, kc, kc[:1], bt, cu, ctx, 0.1), (q, odd, odd, bt, cu, ctx, 0.1), (q[..., :32], small, small, bt, cu, ctx, 0.1),
                 (q, kc, kc, bt, cu, ctx, 0.0), (q, kc, kc, bt, cu, ctx, -1.0), (q, kc, kc, bt[:0], cu, ctx, 0.1), (q, kc, kc, bt, cu[:1], ctx, 0.1), (q, kc.cpu(), kc.cpu(), bt, cu, ctx, 0.1),
                 (q, kc, kc, bt.cpu(), cu, ctx, 0.1), (q, kc.expand(2, 1, -1)[:, :, ::2], kc[:, :, ::2], bt, cu, ctx, 0.1)):
        with pytest.raises(ValueError):
            ops.gqa_attention_paged(*args)
    T = 3
    qkv, rope, slots = torch.zeros(T, 4 * 64, device=DEV, dtype=torch.bfloat16), rope_table(64, 4, DEV), torch.arange(T, device=DEV)
    p1, p3 = torch.zeros(T, dtype=torch.long, device=DEV), torch.zeros(3, T, dtype=torch.long, device=DEV)
    good = dict(qkv=qkv, hd=64, pos=p1, rope=rope, kc=kc, slots=slots, sec=None)
    for bad in (dict(qkv=qkv[:, :-1]), dict(qkv=qkv.float()), dict(pos=p3), dict(pos=p3, sec=[16, 8, 7]), dict(pos=p3[:2], sec=[16, 8, 8]), dict(pos=p3, sec=[]), dict(rope=rope[:, :-2]),
                dict(rope=rope.cpu()), dict(slots=slots[:2]), dict(kc=odd[:, :, :-8]), dict(kc=torch.zeros(2, 16, 1, 64, device=DEV), pos=p3, sec=[16, 8, 8]), dict(pos=p1.cpu())):
        c = {**good, **bad}
        with pytest.raises(ValueError):
            ops.gqa_qkv_prepare(c["qkv"], 2, 1, c["hd"], None, None, 1e-6, False, c["pos"], c["rope"], c["kc"], c["kc"], c["slots"], c["sec"])
    with pytest.raises(ValueError):
        ops.gqa_kv_store(kc, kc, slots, torch.zeros(T, 1, 64, device=DEV), torch.zeros(T, 1, 64, device=DEV))
    one = torch.ones(1, dtype=torch.int32, device=DEV)
    off = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    for kw in (dict(rows=0), dict(rows=2), dict(rows=2, scratch_block=3, pad_len=17), dict(pad_len=0), dict(rows=12001, scratch_block=1)):
        with pytest.raises(ValueError):
            ops.step_tables(one, one, one, off, 16, 1, 1, **kw)
    with pytest.raises(ValueError):
        ops.step_tables(one, one.cpu(), one, off, 16, 1, 1)


def test_empty_calls():
    kc = torch.zeros(2, 1, ops.kv4_page_bytes(64, 16), dtype=torch.uint8, device=DEV)
    none = torch.zeros(0, dtype=torch.long, device=DEV)
    q = ops.gqa_qkv_prepare(torch.zeros(0, 256, device=DEV, dtype=torch.bfloat16), 2, 1, 64, None, None, 1e-6, False, none, rope_table(64, 4, DEV), kc, kc.clone(), none)
    assert q.shape == (0, 2, 64)
    ops.gqa_kv_store(kc, kc, none, q[:, :1], q[:, :1])
    assert ops.gqa_kv_gather(kc, kc, none, 64)[0].shape == (0, 1, 64)
    assert ops.gqa_attention_paged(q, kc, kc, torch.zeros(1, 1, dtype=torch.int32, device=DEV), cu_of([0]), torch.ones(1, dtype=torch.int32, device=DEV), 0.1).shape == (0, 2, 64)
