"""Engines that keep their keys and values in 4 bits: the tokens are those of an engine whose cache holds the same rounded rows in 32 bits, through chunked
prompts, prefix reuse, preemption and the host tier; sizes, page families and refusals."""
import pytest
import torch

from nanoengine_b200 import Config, LLM, SamplingParams, ops
from nanoengine_b200.models.config import ModelConfig, tiny_deepseek_v3, tiny_gemma4, tiny_qwen3_5
from nanoengine_b200.ops import reference as ref
from nanoengine_b200.runtime.cache import KVCache, make_cache_plan

from int4_cases import nearest


def tiny_qwen3(**over):
    base = dict(architecture="Qwen3MoeForCausalLM", vocab_size=512, hidden_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                head_dim=32, intermediate_size=256, n_routed_experts=0, first_k_dense_replace=0, q_lora_rank=None, rope_theta=1e6, max_position_embeddings=4096,
                qk_norm=True, eos_token_id=None)
    base.update(over)
    return ModelConfig(**base)


MODELS = {"qwen3": tiny_qwen3, "qwen3.5": tiny_qwen3_5}


def make(model, kv, **kw):
    base = dict(model="tiny", model_config=MODELS[model](), dummy_weight=True, dtype="float32", device="cpu", kv_cache_dtype=kv, kvcache_block_size=16,
                max_num_seqs=8, num_kvcache_blocks=64, seed=0)
    base.update(kw)
    return LLM(Config(**base))


def prompts(n=4, length=40, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 512, (length + 3 * i,), generator=g).tolist() for i in range(n)]


SP = SamplingParams(temperature=0.0, max_tokens=12, ignore_eos=True)


def tokens(llm):
    return [o["token_ids"] for o in sorted(llm.generate(prompts(), SP), key=lambda o: o["seq_id"])]


@pytest.fixture
def rounded(monkeypatch):
    """The 32-bit cache then holds what the 4-bit one stands for: each row as the nearest of the format's, found in 64 bits."""
    plain = ref.gqa_kv_store

    def store(k_cache, v_cache, slot_mapping, k, v):
        if k_cache.dtype == torch.uint8:
            return plain(k_cache, v_cache, slot_mapping, k, v)
        return plain(k_cache, v_cache, slot_mapping, nearest(k).float(), nearest(v).float())

    monkeypatch.setattr(ref, "gqa_kv_store", store)
    ops.gqa_kv_store                                   # the package keeps what it has dispatched: undone together with the patch
    monkeypatch.setitem(vars(ops), "gqa_kv_store", store)


@pytest.mark.parametrize("model", list(MODELS))
def test_tokens_are_those_of_a_cache_of_rounded_rows(model, rounded):
    # the convolution windows of the second family are kept in bf16 beside 4-bit rows: keep them so in both
    want = None
    for kv in ("float32", "int4"):
        llm = make(model, kv)
        cache = llm.engine.executor.runner.cache
        if cache.conv_states is not None:
            cache.conv_states[:] = [t.float() for t in cache.conv_states]
        got = tokens(llm)
        want = want or got
        assert got == want
    assert cache.kv.dtype == torch.uint8 and int(cache.kv.count_nonzero()) > 0


def test_rounding_shows_in_the_logits():
    """What the cache holds is read back: the logits of a decode step differ from those over unrounded rows, by no more than the rounding explains."""
    outs = []
    for kv in ("float32", "int4"):
        llm = make("qwen3", kv)
        p = prompts(1)[0]
        outs.append(llm.engine.feed([(1, p)], [[len(p) - 1]]))
        llm.engine.end_feed([1])
    a, b = (torch.as_tensor(o) for o in outs)
    assert not torch.equal(a, b) and torch.cosine_similarity(a, b).min() > 0.9


def test_chunks_prefixes_preemption_and_swap_keep_tokens():
    want = tokens(make("qwen3", "int4"))
    assert tokens(make("qwen3", "int4", max_num_batched_tokens=24)) == want
    llm = make("qwen3", "int4")
    assert tokens(llm) == want and tokens(llm) == want                                  # the second run finds its prefixes in the cache
    assert tokens(make("qwen3", "int4", num_kvcache_blocks=14)) == want                 # preempted and recomputed
    assert tokens(make("qwen3", "int4", num_kvcache_blocks=14, num_host_kvcache_blocks=32)) == want


@pytest.mark.parametrize("model", list(MODELS))
def test_sizes_and_page_families(model):
    mc = MODELS[model]()
    plan, wide = (make_cache_plan(mc, kv, 16) for kv in ("int4", "bfloat16"))
    assert plan.kv_block_bytes * 64 == wide.kv_block_bytes * 17 and plan.state_slot_bytes == wide.state_slot_bytes      # 4 bits and a byte per 32: 17 / 64 of bf16
    cache = KVCache(plan, 5, "cpu")
    layers = plan.num_layers
    assert cache.kv.shape == (2, layers, 6, 2, ref.kv4_page_bytes(32, 16)) and cache.kv.numel() == 6 * plan.kv_block_bytes
    fam = cache.page_families()[0]
    assert fam["planes"] == 2 * layers and fam["page_bytes"] * 2 * layers == plan.kv_block_bytes
    cache.kv.copy_(torch.randint(0, 256, cache.kv.shape, dtype=torch.uint8))
    before = cache.kv.clone()
    assert sum(v.numel() for v in cache.block_views(3)) == plan.kv_block_bytes
    cache.allocate_host(2)
    cache.swap([3], [1], to_host=True)
    cache.kv[:, :, 3] = 0
    cache.swap([1], [4], to_host=False)
    assert torch.equal(cache.kv[:, :, 4], before[:, :, 3])


def test_refusals():
    for mc in (tiny_deepseek_v3(), tiny_gemma4(), tiny_qwen3(head_dim=48)):
        with pytest.raises(ValueError, match="int4|4-bit"):
            Config(model="tiny", model_config=mc, dummy_weight=True, dtype="float32", device="cpu", kv_cache_dtype="int4")
    for kw in (dict(dtype="float16"), dict(kvcache_block_size=48), dict(model_config=tiny_qwen3(head_dim=32))):
        with pytest.raises(ValueError, match="4-bit"):
            Config(**dict(dict(model="tiny", model_config=tiny_qwen3(head_dim=64), dummy_weight=True, device="cuda", kv_cache_dtype="int4"), **kw))
    assert Config(model="tiny", model_config=tiny_qwen3(head_dim=64), dummy_weight=True, device="cuda", kv_cache_dtype="int4").kvcache_block_size == 64
    with pytest.raises(ValueError, match="int4"):
        Config(model="tiny", model_config=tiny_qwen3(), dummy_weight=True, device="cpu", kv_cache_dtype="int8")


# ---- image tokens at a time, a row and a column ----------------------------------------------------
IMG = 7
GRIDS = [(1, 4, 6), (2, 2, 4)]                       # patches: 2 x 3 and 2 x (1 x 2) tokens
PROMPT = [3, 11] + [IMG] * 6 + [25, 99, 14] + [IMG] * 4 + list(range(30, 50))


def expected_positions(tokens):
    out, p, i, images = [], 0, 0, [(t, h // 2, w // 2) for t, h, w in GRIDS]
    while i < tokens:
        if i < len(PROMPT) and PROMPT[i] == IMG:
            t, h, w = images.pop(0)
            out += [(p + a, p + b, p + c) for a in range(t) for b in range(h) for c in range(w)]
            i, p = i + t * h * w, p + max(t, h, w)
        else:
            out.append((p, p, p))
            i, p = i + 1, p + 1
    return torch.tensor(out).t()


@pytest.mark.parametrize("kv", ["float32", "int4"])
@pytest.mark.parametrize("kw", [{}, dict(max_num_batched_tokens=16)])
def test_image_tokens_stand_at_time_row_and_column(kv, kw):
    sp = SamplingParams(temperature=0.0, max_tokens=5, ignore_eos=True)
    emb = torch.randn(10, 128, generator=torch.Generator().manual_seed(1)) * 0.02
    seen, text, got = {}, {}, {}
    for grids in (GRIDS, None):
        llm = make("qwen3", kv, enable_prefix_caching=False, model_config=tiny_qwen3(mrope_section=[6, 5, 5], mrope_interleaved=True), **kw)
        runner = llm.engine.executor.runner
        plain = runner.prepare

        def prepare(b, seen=seen, text=text, grids=grids, plain=plain):
            ctx = plain(b)
            lo = 0
            for sid, q, n in zip(b.seq_ids, b.q_lens, b.seq_lens):
                pos = ctx.extras["positions"][:, lo: lo + q]
                (seen if int(sid) == 1 and grids else text).setdefault(int(sid), {})[int(n) - q] = pos.clone()
                lo += q
            return ctx

        runner.prepare = prepare
        llm.engine.add_vision_request(PROMPT, IMG, embeddings=emb, sampling_params=sp, seq_id=1, grid_thw=grids)
        llm.engine.add_request(list(range(60, 90)), sp, seq_id=2)
        got[bool(grids)] = {o["seq_id"]: o["token_ids"] for o in llm.generate()}
        assert not runner._image_axes and not llm.engine._with_axes                # given back when the request is through
    whole = torch.cat([seen[1][k] for k in sorted(seen[1])], 1)
    assert torch.equal(whole, expected_positions(len(PROMPT) + 4))
    for parts in text.values():                                                     # tokens without grids: their index on every axis
        flat = torch.cat([parts[k] for k in sorted(parts)], 1)
        assert torch.equal(flat, torch.arange(flat.shape[1]).expand(3, -1))
    assert got[True][2] == got[False][2]
    if not kw:
        # one step over everything gives the tokens that the cached steps gave
        runner.prepare = plain
        llm = make("qwen3", kv, enable_prefix_caching=False, model_config=tiny_qwen3(mrope_section=[6, 5, 5], mrope_interleaved=True), max_num_batched_tokens=16)
        llm.engine.add_vision_request(PROMPT, IMG, embeddings=emb, sampling_params=sp, seq_id=1, grid_thw=GRIDS)
        assert llm.generate()[0]["token_ids"] == got[True][1]


def test_image_grids_that_do_not_fit_are_refused():
    mc = tiny_qwen3(mrope_section=[6, 5, 5])
    emb = torch.zeros(10, 128)
    llm = make("qwen3", "int4", model_config=mc)
    for grids in ([(1, 4, 6)], [(1, 4, 6), (2, 2, 6)], [(1, 3, 6), (2, 2, 4)], GRIDS + [(1, 2, 2)]):
        with pytest.raises(ValueError):
            llm.engine.add_vision_request(PROMPT, IMG, embeddings=emb, sampling_params=SP, grid_thw=grids)
    assert not llm.engine.executor.runner._image_axes and not llm.engine._with_axes
    seq = llm.engine.add_vision_request(PROMPT, IMG, embeddings=emb, sampling_params=SP, grid_thw=GRIDS)
    assert llm.engine.abort(seq) and not llm.engine.executor.runner._image_axes
    with pytest.raises(ValueError, match="mrope_section"):
        make("qwen3", "int4", model_config=tiny_qwen3(mrope_section=[8, 5, 5]))
    got = ModelConfig.from_dict({"architectures": ["Qwen3ForCausalLM"], "head_dim": 32, "rope_scaling": {"mrope_section": [6, 5, 5], "mrope_interleaved": True}})
    assert got.position_axes == [6, 5, 5] and got.mrope_interleaved
