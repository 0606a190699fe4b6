"""Prompts with images and the prefix cache: pages are shared by prompts whose images and image positions are the same, never by others."""
import pytest
import torch

from nanoengine_b200 import Config, LLM, RequestMigrate, SamplingParams
from nanoengine_b200._native import _core as C
from nanoengine_b200.models.config import ModelConfig
from nanoengine_b200.vl import EmbeddingPool
from nanoengine_b200.vl.encoder_engine import VisionSlot

IMG = 7
PROMPT = list(range(20, 55)) + [IMG] * 64 + list(range(60, 70))          # two pages of text, the images, text
SP = SamplingParams(temperature=0.0, max_tokens=8, ignore_eos=True)
WIDE, TALL = [(1, 4, 64)], [(1, 64, 4)]                                   # 2 x 32 and 32 x 2 tokens


def images(seed):
    return torch.randn(64, 128, generator=torch.Generator().manual_seed(seed)) * 0.5


def make(kv="float32", **kw):
    mc = ModelConfig(architecture="Qwen3MoeForCausalLM", vocab_size=512, hidden_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                     head_dim=32, intermediate_size=256, n_routed_experts=0, first_k_dense_replace=0, q_lora_rank=None, rope_theta=1e6,
                     max_position_embeddings=4096, qk_norm=True, eos_token_id=None, mrope_section=[6, 5, 5], mrope_interleaved=True)
    base = dict(model="tiny", model_config=mc, dummy_weight=True, dtype="float32", device="cpu", kv_cache_dtype=kv, kvcache_block_size=16, max_num_seqs=8,
                num_kvcache_blocks=64, seed=0)
    base.update(kw)
    return LLM(Config(**base))


def ask(llm, emb, grids, prompt=PROMPT, **kw):
    """(the tokens, how many of the prompt's the prefix cache had)"""
    seq = llm.engine.add_vision_request(prompt, IMG, embeddings=emb, sampling_params=SP, grid_thw=grids, **kw)
    first = [t for o in llm.engine.step() for t in o.token_ids]          # the prompt fits one step
    had = llm.engine.scheduler.get(seq).num_cached_prefix
    return first + llm.generate()[0]["token_ids"], had


@pytest.mark.parametrize("kv", ["float32", "int4"])
def test_pages_are_shared_by_the_same_images_at_the_same_places_only(kv):
    cases = [(1, WIDE), (1, TALL), (1, None), (2, WIDE), (1, WIDE)]
    alone = [ask(make(kv), images(i), g)[0] for i, g in cases]
    assert len({tuple(t) for t in alone}) == 4                           # each differs: a page of another one would show
    llm = make(kv)
    got = [ask(llm, images(i), g) for i, g in cases]
    assert [t for t, _ in got] == alone
    assert [n for _, n in got] == [0, 32, 32, 32, 96]                    # the text in front of the images is everybody's, all full pages the last one's


def test_the_same_token_ids_as_text_do_not_see_the_pages_of_images():
    llm = make()
    want = make().generate([PROMPT], SP)[0]["token_ids"]
    with_images, _ = ask(llm, images(1), WIDE)
    assert llm.generate([PROMPT], SP)[0]["token_ids"] == want != with_images
    assert ask(llm, images(1), WIDE) == (with_images, 96)                # nor the other way round


def test_answers_behind_images_are_shared_with_the_next_turn():
    llm = make(kv="int4")
    first, _ = ask(llm, images(1), WIDE)
    longer = PROMPT + first + list(range(80, 95))
    want = ask(make(kv="int4", enable_prefix_caching=False), images(1), WIDE, longer)[0]
    assert ask(llm, images(1), WIDE, longer) == (want, 112)              # 109 + 8 tokens are in the cache, the last one's row is not: seven pages of 16


def test_slots_of_an_encoder_are_told_apart_by_what_they_hold():
    llm = make()
    pool = EmbeddingPool(1, 64, 128, "cpu", torch.float32)
    got = []
    for seed, grids in ((1, WIDE), (2, WIDE), (2, TALL), (1, WIDE)):
        slot = pool.allocate(64)
        pool.write(slot, images(seed))
        seq = llm.engine.add_vision_request(PROMPT, IMG, vision_slot=VisionSlot("e", slot, 64, 128, [list(g) for g in grids]), pool_desc=pool.export(direct=True),
                                            sampling_params=SP)
        llm.engine.step()
        got.append((llm.engine.scheduler.get(seq).num_cached_prefix, llm.generate()[0]["token_ids"]))
        pool.free(slot)
    assert [n for n, _ in got] == [0, 32, 32, 96]
    assert [t for _, t in got] == [ask(make(), images(i), g)[0][1:] for i, g in ((1, WIDE), (2, WIDE), (2, TALL), (1, WIDE))]


def test_preempted_prompts_find_their_own_pages():
    want = [ask(make(enable_prefix_caching=False), images(1), g)[0] for g in (WIDE, TALL)]
    llm = make(num_host_kvcache_blocks=32, num_kvcache_blocks=15)        # room for two prompts of seven pages, not for both answers
    for i, g in enumerate((WIDE, TALL)):
        llm.engine.add_vision_request(PROMPT, IMG, embeddings=images(1), sampling_params=SP, grid_thw=g, seq_id=i + 1)
    assert [o["token_ids"] for o in sorted(llm.generate(), key=lambda o: o["seq_id"])] == want


def test_keys_of_images_travel_with_the_request():
    r = C.RequestIn(3, [1, 2, 3, 4, 5], SP, prefix_keys=[99, 2 ** 64 - 1], prefix_key_at=[1, 4])
    q = C.RequestIn.from_bytes(r.to_bytes())
    assert (q.prefix_keys, q.prefix_key_at) == ([99, 2 ** 64 - 1], [1, 4])
    m = RequestMigrate()
    m.token_ids, m.prompt_len, m.prefix_keys, m.prefix_key_at = [1, 2, 3], 2, [7], [1]
    n = RequestMigrate.from_bytes(m.to_bytes())
    assert (n.prefix_keys, n.prefix_key_at) == ([7], [1])
    llm = make()
    r.prefix_key_at = [1]
    with pytest.raises(ValueError, match="prefix key"):
        llm.engine.add_request_payload(r.to_bytes())
    # a prefill engine hands them on
    llm = make(mode="prefill", model_config=ModelConfig(**dict(llm.engine.config.model_config.__dict__, mrope_section=None)))
    llm.engine.add_vision_request(PROMPT, IMG, embeddings=images(1), sampling_params=SP)
    llm.generate()
    out = llm.engine.export_to_be_migrated()[0]
    assert len(out.prefix_keys) == 1 and out.prefix_key_at == [35]


def test_an_image_in_a_later_turn_keeps_what_the_first_had():
    later = PROMPT + [IMG] * 4 + list(range(80, 95))
    emb, grids = torch.cat([images(1), images(5)[:4]]), WIDE + [(1, 4, 4)]
    want = ask(make(enable_prefix_caching=False), emb, grids, later)[0]
    llm = make()
    first, _ = ask(llm, images(1), WIDE)
    assert ask(llm, emb, grids, later) == (want, 96)                     # six pages in front of the second image
    assert ask(llm, torch.cat([images(1), images(6)[:4]]), grids, later)[1] == 96
    assert ask(llm, emb, grids, later) == (want, 112)                    # 128 tokens, of which seven full pages count


def test_a_refused_request_leaves_the_one_of_its_number_alone():
    want = ask(make(), images(1), WIDE, seq_id=5)[0]
    llm = make()
    llm.engine.add_vision_request(PROMPT, IMG, embeddings=images(1), sampling_params=SP, grid_thw=WIDE, seq_id=5)
    for grids in (TALL, None):
        with pytest.raises(ValueError, match="duplicate"):
            llm.engine.add_vision_request(PROMPT, IMG, embeddings=images(2), sampling_params=SP, grid_thw=grids, seq_id=5)
    assert llm.generate()[0]["token_ids"] == want
    llm = make(max_model_len=64)
    for grids in (WIDE, None):
        with pytest.raises(ValueError, match="max_model_len"):
            llm.engine.add_vision_request(PROMPT, IMG, embeddings=images(1), sampling_params=SP, grid_thw=grids)
    runner = llm.engine.executor.runner
    assert not runner._vision and not runner._image_axes and not llm.engine._with_axes


@pytest.mark.parametrize("axes", [True, False])
@pytest.mark.parametrize("kw", [dict(enable_prefix_caching=False), dict(), dict(max_num_batched_tokens=112)])
def test_preempted_prompts_are_computed_again_with_their_images(axes, kw):
    """Without a host tier a preempted prompt starts over: its image rows have to be there again."""
    grids = [WIDE, TALL] if axes else [None, None]
    want = [ask(make(enable_prefix_caching=False), images(i + 1), g)[0] for i, g in enumerate(grids)]
    llm = make(num_kvcache_blocks=14, **kw)                              # room for two prompts of seven pages, not for the answers
    for i, g in enumerate(grids):
        llm.engine.add_vision_request(PROMPT, IMG, embeddings=images(i + 1), sampling_params=SP, grid_thw=g, seq_id=i + 1)
    preempted, out, runner = 0, {1: [], 2: []}, llm.engine.executor.runner
    while not llm.engine.is_finished():
        for o in llm.engine.step():
            out[o.seq_id] += o.token_ids
        preempted += sum(v.num_preemptions for v in map(llm.engine.scheduler.get, (1, 2)) if v is not None)
    assert preempted and [out[1], out[2]] == want
    assert not runner._vision and not runner._image_axes and not llm.engine._with_axes


@pytest.mark.parametrize("kv", ["float32", "int4"])
@pytest.mark.parametrize("slot", [True, False])
def test_prefill_and_decode_engines_place_images_like_one_engine(kv, slot):
    """The prompt's rows are turned on the prefill engine, what follows goes on behind the images on the decode engine."""
    from nanoengine_b200.parallel.kv_transfer import KVMigrator, LocalTransport
    cases = [(1, WIDE), (2, TALL), (3, None)]
    want = [ask(make(kv), images(i), g)[0] for i, g in cases]
    prefill, decode = make(kv, mode="prefill", engine_id="p0"), make(kv, mode="decode", engine_id="d0")
    decode.engine.migrator = KVMigrator(LocalTransport([prefill.engine.executor.runner], [decode.engine.executor.runner]), decode.engine.engine_info(),
                                        prefill.engine.engine_info())
    pool = EmbeddingPool(3, 64, 128, "cpu", torch.float32)
    for i, g in cases:
        if slot:
            s = pool.allocate(64)
            pool.write(s, images(i))
            kw = dict(vision_slot=VisionSlot("e", s, 64, 128, [list(x) for x in g or []]), pool_desc=pool.export(direct=True))
        else:
            kw = dict(embeddings=images(i), grid_thw=g)
        prefill.engine.add_vision_request(PROMPT, IMG, sampling_params=SP, seq_id=i, **kw)
    blobs = prefill.generate(return_serialized=True)
    assert not prefill.engine.executor.runner._vision and not prefill.engine._with_axes
    first = {}
    for b in blobs:
        sid, tok = RequestMigrate.from_bytes(b).metadata
        first[sid] = tok
        decode.add_request_payload(b)
    got = {o["seq_id"]: [first[o["seq_id"]]] + o["token_ids"] for o in decode.generate()}
    assert [got[i] for i, _ in cases] == want
    assert not decode.engine.executor.runner._image_axes and not decode.engine._with_axes
    # a hand-over that fails leaves nothing either
    decode.engine.migrator.fail_next = True
    prefill.engine.add_vision_request(PROMPT, IMG, embeddings=images(1), sampling_params=SP, seq_id=9, grid_thw=WIDE)
    decode.add_request_payload(prefill.generate(return_serialized=True)[-1])
    assert decode.generate() == [] and not decode.engine.executor.runner._image_axes and not decode.engine._with_axes


def test_images_under_pipeline_stages_are_refused(monkeypatch):
    llm = make(mode="prefill")
    monkeypatch.setattr(llm.engine.config, "pp", 2)
    with pytest.raises(ValueError, match="pipeline"):
        llm.engine.add_vision_request(PROMPT, IMG, embeddings=images(1), sampling_params=SP, grid_thw=WIDE)
    assert not llm.engine._with_axes and llm.engine.scheduler.num_waiting() == 0


def test_a_prompt_that_no_engine_has_run_stands_at_its_index():
    """Only a hand-over says how far tokens stand from their index; a prompt of its own is placed by its images."""
    want = make().generate([PROMPT], SP)[0]["token_ids"]
    llm = make()
    llm.engine.add_request_payload(C.RequestIn(1, PROMPT, SP, position_shift=9).to_bytes())
    assert not llm.engine._with_axes and llm.generate()[0]["token_ids"] == want


def test_images_with_speculative_decoding():
    """Prompts of an engine that drafts splice the image rows in like those of others."""
    from nanoengine_b200.models.config import tiny_deepseek_v3
    got = []
    for spec in (0, 2):
        mc = tiny_deepseek_v3()
        mc.num_nextn_predict_layers = 1
        llm = LLM(Config(model="tiny-deepseek-v3", model_config=mc, dummy_weight=True, dtype="float32", device="cpu", kvcache_block_size=16, num_kvcache_blocks=32,
                         max_num_seqs=4, num_speculative_tokens=spec, seed=0))
        for seed in (1, 2):
            emb = torch.randn(6, mc.hidden_size, generator=torch.Generator().manual_seed(seed)) * 0.5
            llm.engine.add_vision_request([3, 11] + [IMG] * 6 + list(range(30, 60)), IMG, embeddings=emb, sampling_params=SP, seq_id=seed)
        got.append([o["token_ids"] for o in sorted(llm.generate(), key=lambda o: o["seq_id"])])
    assert got[0] == got[1] and got[0][0] != got[0][1]
