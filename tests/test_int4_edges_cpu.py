"""4-bit pages, positions on several axes and step tables: calls at the edges of what the operators allow."""
import pytest
import torch

from nanoengine_b200 import ops


def overlapping(device):
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device=device)                 # noqa: E731
    i64 = lambda n: torch.zeros(n, dtype=torch.int64, device=device)                 # noqa: E731
    new, ctx, ids, off = (torch.tensor(t, dtype=torch.int32, device=device) for t in ([1, 1], [5, 40], [3, 1, 2], [0, 1, 3]))
    for table in (i32(4).expand(2, 4), i32(6).as_strided((2, 4), (1, 1)), i32(2).expand(2, 2)):
        out = ops.StepTables(i32(3), i32(2), i64(2), i64(2), table, i32(2))
        with pytest.raises(ValueError, match="overlap"):
            ops.step_tables(new, ctx, ids, off, 32, 2, 2, out=out)
        assert not table.any()
    # one row may have any stride
    out = ops.StepTables(i32(2), i32(1), i64(1), i64(1), i32(4).expand(1, 4), i32(1))
    got = ops.step_tables(new[:1], ctx[1:], ids[1:], off[:2] * 2, 32, 1, 2, out=out)
    assert got.block_tables.tolist() == [[1, 2]] and got.slot_mapping.tolist() == [71]


def test_tables_whose_rows_overlap_are_refused():
    overlapping("cpu")


@pytest.mark.parametrize("sections,interleaved", [([48], False), ([16, 16, 16], True), ([20, 0, 28], False), ([24, 16, 8], True), ([10, 12, 14, 12], False), ([4, 30, 7, 7], True)])
def test_rows_of_angles_by_axis(sections, interleaved):
    """What the GPU's separate kernels turn rows by is the plain form's table."""
    from nanoengine_b200.ops import reference as ref, sm100
    g = torch.Generator().manual_seed(1)
    table, pos = torch.randn(50, 96, generator=g), torch.randint(0, 50, (len(sections), 9), generator=g)
    assert torch.equal(sm100._axes_table(pos, table, sections, interleaved, 9, 96), ref.rope_axes_rows(pos, table, sections, interleaved))
    with pytest.raises(ValueError, match="sections"):
        sm100._axes_table(pos, table, [47], interleaved, 9, 96)
    with pytest.raises(ValueError, match="one row per axis"):
        sm100._axes_table(pos[:, :8], table, sections, interleaved, 9, 96)


@pytest.mark.parametrize("hq,hkv,dim", [(64, 4, 128), (32, 8, 128), (16, 2, 256), (8, 1, 64), (8, 8, 128), (9, 3, 64)])
def test_no_step_expands_more_than_its_engine_leaves_free(hq, hkv, dim, monkeypatch):
    """Every step that an engine can be asked for: tokens, sequences and widths up to its limits."""
    from nanoengine_b200.ops import sm100, sm100_attn
    asked = []

    class Expanded(Exception):
        pass

    def expand(k, v, bt, cl, d):
        asked.append(4 * cl.numel() * -(-bt.shape[1] * sm100.kv4_block_size(k, d) // 64) * 64 * hkv * d)
        raise Expanded

    class Kernel(Exception):
        pass

    def kernel(*a):
        raise Kernel

    monkeypatch.setattr(sm100, "kv4_expand", expand)
    monkeypatch.setattr(sm100, "_same_device", lambda *a: None)
    monkeypatch.setattr(sm100_attn, "_INT4_SHARES", {(d, r): 8 for d in (64, 128, 256) for r in (8, 16)})
    monkeypatch.setattr(sm100_attn, "_sms", kernel)                      # the other kernel's way begins here
    most_seen = 0
    for bs in (16, 64, 256):
        for tokens, seqs, length in ((512, 8, 4096), (8192, 64, 32768), (2048, 2, 131072)):
            room = sm100_attn.int4_expansion_room(tokens, seqs, length, hq, hkv, dim, bs)
            kc = torch.zeros(1, hkv, sm100.kv4_page_bytes(dim, bs), dtype=torch.uint8)
            for B in {1, 2, seqs // 2, seqs}:
                for T in {B, 4 * B, 16 * B, 64 * B, 512 * B, tokens}:
                    for W in {1, 2, length // bs // 2, length // bs, length // bs + 1}:
                        if B <= T <= tokens and W:
                            q = torch.empty(T, hq, dim, dtype=torch.bfloat16, device="meta")
                            with pytest.raises((Expanded, Kernel)):
                                sm100_attn._gqa_int4(q, kc, kc, torch.empty(B, W, dtype=torch.int32, device="meta"), torch.empty(B + 1, dtype=torch.int32, device="meta"),
                                                     torch.empty(B, dtype=torch.int32, device="meta"), 0.1, 0)
            most_seen = max(most_seen, max(asked, default=0))
            assert all(n <= room for n in asked) and room <= 2 << 30
            asked.clear()
    assert (most_seen > 0) == (hq // hkv % 4 == 0 or hq == hkv)
