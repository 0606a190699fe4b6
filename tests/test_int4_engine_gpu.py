"""Engines over a 4-bit cache on the GPU: captured and eager steps agree, the logits are those of the CPU's engine, a step's tables built on the device
are the host's."""
import pytest
import torch

from nanoengine_b200 import Config, LLM, SamplingParams
from nanoengine_b200._native import _core as C
from nanoengine_b200.models.config import ModelConfig, tiny_qwen3_5

pytestmark = pytest.mark.gpu

IMG = 7


def small(**over):
    base = dict(architecture="Qwen3MoeForCausalLM", vocab_size=512, hidden_size=256, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=2,
                head_dim=64, intermediate_size=512, n_routed_experts=0, first_k_dense_replace=0, q_lora_rank=None, rope_theta=1e6, max_position_embeddings=4096,
                qk_norm=True, eos_token_id=None)
    base.update(over)
    return ModelConfig(**base)


def make(mc, kv="int4", device="cuda", **kw):
    base = dict(model="small", model_config=mc, dummy_weight=True, dtype="bfloat16" if device == "cuda" else "float32", device=device, kv_cache_dtype=kv,
                kvcache_block_size=16, max_num_seqs=8, num_kvcache_blocks=128, max_model_len=512, seed=0)
    base.update(kw)
    return LLM(Config(**base))


def prompts(lens, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(8, 512, (n,), generator=g).tolist() for n in lens]


SP = SamplingParams(temperature=0.0, max_tokens=10, ignore_eos=True)


@pytest.mark.parametrize("lens", [(1, 40, 17), (5,), (33, 64, 2, 100, 129)])
def test_step_inputs_are_those_of_the_host(lens):
    llm = make(small(), enforce_eager=True)
    runner = llm.engine.executor.runner
    bs = 16
    for new in (0, 1, 3):                                       # whole prompts, one new token, three
        b = C.RunnerIn()
        q = [min(n, new) if new else n for n in lens]
        pages = [-(-n // bs) for n in lens]
        b.is_prefill, b.seq_ids, b.q_lens, b.seq_lens = not new, list(range(len(lens))), q, list(lens)
        b.positions = [p for n, k in zip(lens, q) for p in range(n - k, n)]
        b.input_ids = [(7 * i) % 512 for i in range(sum(q))]
        perm = torch.randperm(128, generator=torch.Generator().manual_seed(1)).tolist()
        b.block_tables, b.block_offsets = perm[: sum(pages)], [sum(pages[:i]) for i in range(len(lens) + 1)]
        b.temperatures, b.sample_mask = [0.0] * len(lens), [1] * len(lens)
        b.state_slots = b.handoff_slots = b.hisparse_slots = [-1] * len(lens)
        ctx, want = runner.prepare(b), b.prepare(bs, 0)
        assert ctx.extras["tables_of"] is not None
        got = dict(cu_seqlens_q=ctx.cu_seqlens_q, context_lens=ctx.context_lens, slot_mapping=ctx.slot_mapping, block_tables=ctx.block_tables.reshape(-1),
                   last_token_indices=ctx.last_token_indices, input_ids=ctx.extras["input_ids"], positions=ctx.extras["positions"])
        for name, t in got.items():
            assert torch.equal(t.cpu().long(), torch.as_tensor(want[name]).long()), name
        assert ctx.max_seqlen_q == want["max_seqlen_q"] and ctx.max_seqlen_k == want["max_seqlen_k"]
        b.positions = [p + (1 if i == 0 else 0) for i, p in enumerate(b.positions)] if lens[0] % bs else b.positions
        if lens[0] % bs:                                        # a token that does not stand where the lengths put it: the host's tables
            ctx, want = runner.prepare(b), b.prepare(bs, 0)
            assert ctx.extras["tables_of"] is None and torch.equal(ctx.slot_mapping.cpu(), torch.as_tensor(want["slot_mapping"]))
    with pytest.raises(RuntimeError, match="beyond"):
        b.positions = [4000] * len(b.positions)
        runner.prepare(b)


AXES = dict(num_key_value_heads=8, head_dim=128, mrope_section=[24, 20, 20], mrope_interleaved=True)


# bf16 pages of the third want four query heads per kv head on the GPU
@pytest.mark.parametrize("mc,kv", [(small(), "int4"), (small(), "auto"), (small(**AXES), "int4"), (small(**AXES), "auto"),
                                   (tiny_qwen3_5(head_dim=64, num_attention_heads=4), "int4")], ids=["qwen3-4", "qwen3", "axes-4", "axes", "qwen3.5-4"])
def test_captured_steps_are_the_eager_ones(mc, kv):
    ps = prompts((40, 17, 130, 64, 3))
    got = []
    for eager in (True, False):
        llm = make(mc, kv, enforce_eager=eager)
        got.append([o["token_ids"] for o in sorted(llm.generate(ps, SP), key=lambda o: o["seq_id"])])
        if not eager:
            assert llm.engine.executor.runner.graph_step_equals_eager()
    assert got[0] == got[1]


def test_logits_are_those_of_the_cpu():
    """Prompt, then three single tokens, then five at once, next to the 32-bit engine over rows rounded the same way.  The GPU's activations are bf16: each of
    the two layers rounds a handful of times at 2^-8 and a flipped code moves a row by a seventh of its largest value, so the logits agree in direction."""
    from nanoengine_b200.ops import sm100_attn
    p = prompts((70,))[0]
    outs = []
    for device in ("cuda", "cpu"):
        before = sm100_attn.INT4_CALLS[0]
        llm, rows = make(small(), device=device), []
        model = llm.engine.executor.runner.model
        if device == "cuda":                                    # random weights are drawn on the engine's device: the second engine takes the first one's
            weights = {n: t.detach().float().cpu() for n, t in model.named_parameters()}
        else:
            for n, t in model.named_parameters():
                t.data.copy_(weights.pop(n))
            assert not weights
        rows.append(llm.engine.feed([(1, p)], [[0, 30, 69]]))
        for t in (11, 12, 13):
            rows.append(llm.engine.feed([(1, [t])], [[0]]))
        rows.append(llm.engine.feed([(1, [20, 21, 22, 23, 24])], [[0, 4]]))
        llm.engine.end_feed([1])
        outs.append(torch.cat([torch.as_tensor(r) for r in rows]))
        assert (sm100_attn.INT4_CALLS[0] > before) == (device == "cuda")
    assert torch.cosine_similarity(outs[0], outs[1]).min() > 0.99


def test_images_over_three_axes_captured_and_eager():
    mc = small(**AXES)
    prompt = [30, 11] + [IMG] * 6 + [25, 99, 14] + [IMG] * 4 + list(range(30, 50))
    emb = torch.randn(10, 256, generator=torch.Generator().manual_seed(1)) * 0.02
    got = []
    for kw in (dict(enforce_eager=True), {}, dict(max_num_batched_tokens=16)):
        llm = make(mc, enable_prefix_caching=False, **kw)
        llm.engine.add_vision_request(prompt, IMG, embeddings=emb, sampling_params=SP, seq_id=1, grid_thw=[(1, 4, 6), (2, 2, 4)])
        llm.engine.add_request(prompts((50,))[0], SP, seq_id=2)
        got.append({o["seq_id"]: o["token_ids"] for o in llm.generate()})
        assert not llm.engine.executor.runner._image_axes
    assert got[0] == got[1]
    assert len(got[2][1]) == len(got[0][1]) == 10            # in chunks the sums of the prompt's rows are rounded in another order


def test_host_tier_brings_pages_back():
    mc, ps = small(), prompts((60, 61, 62, 63))

    llm = make(mc, num_kvcache_blocks=18, num_host_kvcache_blocks=64)
    assert [len(o["token_ids"]) for o in llm.generate(ps, SP)] == [10] * 4
    cache = llm.engine.executor.runner.cache
    before = cache.kv[:, :, 2].clone()
    cache.swap([2], [1], to_host=True)
    cache.kv[:, :, 2] = 0
    cache.swap([1], [3], to_host=False)
    torch.cuda.synchronize()
    assert torch.equal(cache.kv[:, :, 3], before) and int(before.count_nonzero())
