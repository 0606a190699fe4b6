"""4-bit key / value rows, positions on several axes and the step tables: the plain statements against 64 bits and against the host's own tables."""
import pytest
import torch

from int4_cases import LEVELS, attention_bound, axis_of, cache_values, decode_row, dense_attention, level, nearest, random_cache, rope_table, rows_exact, softmax_scale, table_of, tables_exact
from nanoengine_b200 import ops
from nanoengine_b200._native import _core as C
from nanoengine_b200.ops import reference as ref


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def test_every_scale_byte_is_finite_and_exact_in_bf16():
    assert all(LEVELS[b] < LEVELS[b + 1] for b in range(255)) and float(LEVELS[0]) == 2.0 ** -16 and float(LEVELS[255]) == 1.875 * 2 ** 15
    codes = torch.arange(16, dtype=torch.float64) - 8
    every = torch.outer(LEVELS, codes)
    assert torch.equal(every.to(torch.bfloat16).to(torch.float64), every)


@pytest.mark.parametrize("dim", [32, 64, 96, 128, 256])
def test_quantised_rows_are_the_nearest_and_read_back_byte_by_byte(dim):
    g = gen(dim)
    x = (torch.randn(6, 3, dim, generator=g) * torch.exp2(torch.randint(-14, 13, (6, 3, dim // 32), generator=g).float()).repeat_interleave(32, -1)).to(torch.bfloat16)
    codes, scales = ref.kv4_quant(x)
    got = ref.kv4_values(codes, scales).double()
    assert torch.equal(got, nearest(x))
    row = bytes(codes[2, 1].tolist()) + bytes(scales[2, 1].tolist())
    assert decode_row(row, 0, dim, 1) == got[2, 1].tolist()
    s = LEVELS[scales.long()].repeat_interleave(32, -1)
    assert bool(((x.double() - got).abs() <= s / 2).all())


def test_borders_extremes_and_non_numbers_of_the_format():
    # a seventh of 119 / 16 lies midway between two scales: the even one; so does a code midway between two multiples
    assert ref.kv4_quant(torch.tensor([[119 / 16] + [0.0] * 31]))[1].item() % 2 == 0
    x = torch.zeros(1, 32)
    x[0, :4] = torch.tensor([7.0, 0.5, 1.5, 2.5])
    assert ref.kv4_values(*ref.kv4_quant(x))[0, :4].tolist() == [7.0, 0.0, 2.0, 2.0]
    most = 7 * level(255)
    x[0, :4] = torch.tensor([float("inf"), -float("inf"), float("nan"), 1e30])
    assert ref.kv4_values(*ref.kv4_quant(x))[0, :4].tolist() == [most, -most, 0.0, most]
    assert ref.kv4_values(*ref.kv4_quant(torch.full((1, 32), float("nan")))).abs().sum() == 0
    assert ref.kv4_values(*ref.kv4_quant(torch.zeros(2, 64))).abs().sum() == 0
    tiny = torch.full((1, 32), 2.0 ** -17)
    assert set(ref.kv4_values(*ref.kv4_quant(tiny))[0].tolist()) <= {0.0, 2.0 ** -16}
    for byte in (0, 0x7F, 0x80, 0xFF):
        assert torch.isfinite(ref.kv4_values(torch.full((1, 16), byte, dtype=torch.uint8), torch.full((1, 1), byte, dtype=torch.uint8))).all()


@pytest.mark.parametrize("bs", [1, 16, 64])
def test_store_and_gather_touch_their_slots_only(bs):
    g = gen(3)
    hkv, dim, blocks, T = 2, 64, 7, 5
    kc, vc = (torch.full((blocks, hkv, ops.kv4_page_bytes(dim, bs)), 0xAB, dtype=torch.uint8) for _ in range(2))
    k, v = (torch.randn(T, hkv, dim, generator=g).to(torch.bfloat16) for _ in range(2))
    slots = torch.tensor([blocks * bs - 1, -1, 0, 3, blocks * bs])          # padding, and a slot behind the cache
    before = cache_values(kc, dim)
    ops.gqa_kv_store(kc, vc, slots, k, v)
    a, b = ops.gqa_kv_gather(kc, vc, slots, dim)
    for got, x in ((a, k), (b, v)):
        want = nearest(x)
        want[1] = want[4] = 0
        assert got.dtype == torch.bfloat16 and torch.equal(got.double(), want)
    after = cache_values(kc, dim).flatten(0, 1)
    same = torch.ones(blocks * bs, dtype=torch.bool)
    same[[blocks * bs - 1, 0, 3]] = False
    assert torch.equal(after[same], before.flatten(0, 1)[same])


@pytest.mark.parametrize("sections,interleaved", [([4, 6, 6], False), ([8, 4, 4], True), ([6, 6, 4], True), ([16], False), ([0, 16], False), ([5, 4, 4, 3], False), ([2, 7, 7], True)])
@pytest.mark.parametrize("int4", [False, True])
def test_rows_with_a_position_per_axis(sections, interleaved, int4):
    g = gen(5)
    T, hq, hkv, d, bs = 9, 4, 2, 32, 16
    qkv = torch.randn(T, (hq + 2 * hkv) * d, generator=g)
    qw, kw = torch.rand(d, generator=g) + 0.5, torch.rand(d, generator=g) + 0.5
    pos = torch.randint(0, 50, (len(sections), T), generator=g)
    table = rope_table(d, 50)
    kc, vc = (torch.zeros(3, hkv, ops.kv4_page_bytes(d, bs), dtype=torch.uint8) if int4 else torch.zeros(3, bs, hkv, d) for _ in range(2))
    slots = torch.randperm(3 * bs, generator=g)[:T]
    q = ops.gqa_qkv_prepare(qkv, hq, hkv, d, qw, kw, 1e-6, True, pos, table, kc, vc, slots, sections, interleaved)
    x = qkv.view(T, -1, d)
    want_q = rows_exact(x[:, :hq], qw, 1e-6, 1.0, pos, table, sections, interleaved)
    want_k = rows_exact(x[:, hq: hq + hkv], kw, 1e-6, 1.0, pos, table, sections, interleaved)
    assert (q.double() - want_q).abs().max() <= 2.0 ** -20 * want_q.abs().max()
    if int4:
        k, v = ops.gqa_kv_gather(kc, vc, slots, d)
        assert torch.equal(k.double(), nearest(want_k)) and torch.equal(v.double(), nearest(x[:, hq + hkv:]))
    else:
        assert (kc.view(-1, hkv, d)[slots].double() - want_k).abs().max() <= 2.0 ** -20 * want_k.abs().max()
        assert torch.equal(vc.view(-1, hkv, d)[slots], x[:, hq + hkv:])


def test_equal_positions_on_all_axes_are_ordinary_positions():
    g = gen(6)
    T, d = 7, 64
    qkv, pos, table = torch.randn(T, 4 * d, generator=g), torch.randint(0, 90, (T,), generator=g), rope_table(64, 90)
    made = []
    for p, sec in ((pos, None), (pos.expand(3, T), [12, 10, 10])):
        kc, vc = (torch.zeros(2, 1, ops.kv4_page_bytes(d, 16), dtype=torch.uint8) for _ in range(2))
        made.append((ops.gqa_qkv_prepare(qkv, 2, 1, d, None, None, 1e-6, False, p, table, kc, vc, torch.arange(T), sec), kc, vc))
    assert all(torch.equal(a, b) for a, b in zip(*made))


def test_axes_of_the_angles():
    for half, sections, inter in ((64, [16, 24, 24], False), (64, [24, 20, 20], True), (64, [16, 24, 24], True), (16, [1, 15], True)):
        assert ref.angle_axes(half, sections, inter).tolist() == [axis_of(i, sections, inter) for i in range(half)]
    for half, sections in ((64, [16, 24, 23]), (64, [65, -1]), (10, [2, 2, 2, 2, 2]), (4, [])):
        with pytest.raises(ValueError):
            ref.angle_axes(half, sections, False)


ATTENTION = [
    # hq, hkv, dim, block size, new tokens, contexts, window
    (4, 1, 64, 16, [1, 1, 1], [1, 16, 17], 0),
    (8, 2, 64, 64, [3, 1, 0, 5], [3, 70, 9, 64], 0),
    (6, 2, 32, 4, [2, 4], [9, 4], 3),
    (2, 2, 128, 32, [1], [100], 1),
    (3, 1, 96, 8, [5], [3], 0),                                        # more new tokens than context: the first see nothing
    (4, 2, 64, 16, [1, 1], [0, 40], 0),
]


@pytest.mark.parametrize("hq,hkv,dim,bs,new,ctx,window", ATTENTION)
def test_attention_over_4_bit_pages(hq, hkv, dim, bs, new, ctx, window):
    g = gen(7)
    table, _, _ = table_of(ctx, bs, 40, g)
    kc, vc = (random_cache(40, hkv, dim, bs, g) for _ in range(2))
    q = torch.randn(sum(new), hq, dim, generator=g)
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32)
    got = ops.gqa_attention_paged(q, kc, vc, table, cu, torch.tensor(ctx, dtype=torch.int32), softmax_scale(dim), window)
    out, spread, mass, top = dense_attention(q, cache_values(kc, dim), cache_values(vc, dim), table, new, ctx, softmax_scale(dim), window)
    assert bool(((got.double() - out).abs() <= attention_bound(out, spread, mass, top)).all())


def test_pages_outside_the_cache_read_as_zeros_and_contexts_end_with_their_tables():
    g = gen(8)
    kc, vc = (random_cache(5, 1, 64, 16, g) for _ in range(2))
    table = torch.tensor([[2, -1, 4], [5, 1, 0]], dtype=torch.int32)
    q = torch.randn(2, 2, 64, generator=g)
    cu, ctx = torch.tensor([0, 1, 2], dtype=torch.int32), torch.tensor([40, 1000], dtype=torch.int32)
    got = ops.gqa_attention_paged(q, kc, vc, table, cu, ctx, 0.1)
    out, spread, mass, top = dense_attention(q, cache_values(kc, 64), cache_values(vc, 64), table, [1, 1], [40, 1000], 0.1)
    assert bool(((got.double() - out).abs() <= attention_bound(out, spread, mass, top)).all())


def test_refusals_of_caches_that_do_not_fit():
    kc = torch.zeros(2, 1, ops.kv4_page_bytes(64, 16), dtype=torch.uint8)
    q, cu, ctx, bt = torch.zeros(1, 2, 64), torch.tensor([0, 1]), torch.tensor([1]), torch.zeros(1, 1, dtype=torch.int32)
    for bad in (kc[:, :, :-1], kc.view(2, -1), kc.expand(2, 3, -1)):
        with pytest.raises(ValueError):
            ops.gqa_attention_paged(q, bad, bad, bt, cu, ctx, 0.1)
    with pytest.raises(ValueError):
        ops.gqa_attention_paged(q, kc, kc[:1], bt, cu, ctx, 0.1)
    with pytest.raises(ValueError):
        ops.kv4_page_bytes(48, 16)
    with pytest.raises(ValueError):
        ops.kv4_quant(torch.zeros(1, 40))
    args = (torch.zeros(3, 4 * 64), 2, 1, 64, None, None, 1e-6, False)
    rope, slots = rope_table(64, 4), torch.arange(3)
    for pos, sec in ((torch.zeros(2, 3, dtype=torch.long), [16, 8, 8]), (torch.zeros(3, 3, dtype=torch.long), [16, 8, 7]), (torch.zeros(3, dtype=torch.long), [16, 8, 8])):
        with pytest.raises(ValueError):
            ops.gqa_qkv_prepare(*args, pos, rope, kc, kc.clone(), slots, sec)


TABLES = [
    # block size, new, ctx, rows, padding, tokens beyond, columns beyond
    (64, [1, 1, 1], [1, 64, 65], 3, 1, 0, 0),
    (64, [1, 1, 1], [1, 64, 65], 8, 1, 0, 2),
    (16, [5, 0, 20], [5, 9, 33], 4, 3, 6, 0),
    (1, [2, 3], [7, 3], 2, 1, 0, 1),
    (64, [300], [1000], 1, 1, 0, 0),
    (32, [], [], 2, 2, 1, 1),
    (32, [], [], 0, 1, 3, 0),
]


@pytest.mark.parametrize("bs,new,ctx,rows,pad,extra,wide", TABLES)
def test_step_tables_against_loops(bs, new, ctx, rows, pad, extra, wide):
    table, ids, off = table_of(ctx, bs, 300 if bs > 1 else 40, gen(1))
    width, tokens = table.shape[1] + wide, sum(new) + (rows - len(new)) * pad + extra
    got = ops.step_tables(torch.tensor(new, dtype=torch.int32), torch.tensor(ctx, dtype=torch.int32), ids, off, bs, tokens, width, rows, pad, 999)
    want = tables_exact(new, ctx, ids.tolist(), off.tolist(), bs, tokens, width, rows, pad, 999)
    for name, a, b in zip(got._fields, got, want):
        assert a.dtype == b.dtype and torch.equal(a, b), name


def test_step_tables_of_bad_lengths_and_pages_store_nothing():
    new, ctx, bs = [3, 2, 4], [1, 40, 100], 16
    ids, off = torch.tensor([4, -7, 2, 9], dtype=torch.int32), torch.tensor([0, 1, 3, 9], dtype=torch.int32)       # page -7; an offset behind the list; too few pages
    got = ops.step_tables(torch.tensor(new, dtype=torch.int32), torch.tensor(ctx, dtype=torch.int32), ids, off, bs, 9, 3)
    want = tables_exact(new, ctx, ids.tolist(), off.tolist(), bs, 9, 3, 3, 1, -1)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert got.slot_mapping.tolist() == [-1, -1, 64, -1, -1, -1, -1, -1, -1]


def test_step_tables_write_the_front_of_larger_buffers():
    new, ctx, bs = [1, 2], [5, 40], 16
    table, ids, off = table_of(ctx, bs, 9, gen(2))
    big = ops.StepTables(*(torch.full(s, -5, dtype=t) for s, t in (((9,), torch.int32), ((8,), torch.int32), ((11,), torch.int64), ((11,), torch.int64),
                                                                    ((8, 7), torch.int32), ((8,), torch.int32))))
    got = ops.step_tables(torch.tensor(new, dtype=torch.int32), torch.tensor(ctx, dtype=torch.int32), ids, off, bs, 4, 3, 3, 1, 8, out=big)
    want = tables_exact(new, ctx, ids.tolist(), off.tolist(), bs, 4, 3, 3, 1, 8)
    for a, b, whole in zip(got, want, big):
        assert torch.equal(a, b) and a.data_ptr() == whole.data_ptr()
        left = whole.clone()
        left[tuple(slice(k) for k in b.shape)] = -5
        assert bool((left == -5).all())
    for short in range(6):
        bad = list(big)
        bad[short] = bad[short][:2]
        with pytest.raises(ValueError):
            ops.step_tables(torch.tensor(new, dtype=torch.int32), torch.tensor(ctx, dtype=torch.int32), ids, off, bs, 4, 3, 3, 1, 8, out=ops.StepTables(*bad))


def test_step_tables_refusals():
    one = torch.ones(1, dtype=torch.int32)
    off = torch.tensor([0, 1], dtype=torch.int32)
    for kw in (dict(rows=0), dict(rows=2), dict(rows=2, scratch_block=3, pad_len=17), dict(pad_len=0)):
        with pytest.raises(ValueError):
            ops.step_tables(one, one, one, off, 16, 1, 1, **kw)
    for args in ((one, one, one, off, 0, 1, 1), (one, one, one, off, 16, -1, 1), (one, one, one, off, 16, 1, 0), (one, torch.ones(2), one, off, 16, 1, 1), (one, one, one, one, 16, 1, 1)):
        with pytest.raises(ValueError):
            ops.step_tables(*args)


def test_step_tables_are_the_host_tables():
    """The C++ preparation of a batch makes the same tables."""
    b = C.RunnerIn()
    b.is_prefill = True
    new, ctx, bs = [3, 1, 17], [3, 40, 50], 16
    table, ids, off = table_of(ctx, bs, 30, gen(9))
    b.seq_ids, b.q_lens, b.seq_lens = [0, 1, 2], new, ctx
    b.input_ids = [1] * sum(new)
    b.positions = [p for n, c in zip(new, ctx) for p in range(c - n, c)]
    b.block_tables, b.block_offsets = ids.tolist(), off.tolist()
    b.temperatures, b.sample_mask = [0.0] * 3, [1] * 3
    d = b.prepare(bs, 0)
    got = ops.step_tables(torch.tensor(new), torch.tensor(ctx), ids, off, bs, sum(new), int(d["max_blocks"]))
    for name in got._fields:
        assert torch.equal(getattr(got, name).flatten().long(), torch.from_numpy(d[name]).flatten().long()), name


@pytest.mark.parametrize("dim,bs,fits", [(32, 1, False), (32, 2, False), (32, 3, False), (32, 4, True), (32, 6, False), (64, 1, False), (64, 2, True), (64, 3, False),
                                         (128, 1, True), (128, 3, True), (256, 1, True)])
def test_the_gpu_takes_pages_of_whole_words_only(dim, bs, fits):
    """The kernels move words of eight codes; the check is the host's and needs no GPU."""
    from nanoengine_b200.ops import sm100
    cache = torch.zeros(4, 2, ops.kv4_page_bytes(dim, bs), dtype=torch.uint8)
    if fits:
        assert sm100._kv4_dims(cache, cache, 2, dim) == bs
    else:
        with pytest.raises(ValueError, match="whole words"):
            sm100._kv4_dims(cache, cache, 2, dim)
