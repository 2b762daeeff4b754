"""The engine over the 4-bit KV cache, with and without a cache budget, and int8 projections."""

import pytest
import torch

from afd_plugin_b200.engine_config import CacheConfig, EngineConfig, ModelConfig
from afd_plugin_b200.models import build_model, get_preset
from afd_plugin_b200.models.layers import Int4Layer
from afd_plugin_b200.runtime.engine import LLMEngine
from afd_plugin_b200.runtime.kv_cache import KVCache

PROMPTS = [[(7 * i + j * j) % 250 for j in range(n)] for i, n in enumerate((37, 5, 70, 1))]


def _engine(preset="tiny-qwen3-moe", arch_kw=None, chunk=None, async_scheduling=False, num_blocks=None, **cache):
    arch = get_preset(preset).scaled(**(arch_kw or {}))
    cc = CacheConfig(**{"block_size": 16, "num_blocks": num_blocks, "kv_cache_dtype": "int4", **cache})
    ec = EngineConfig(ModelConfig(arch, dtype=torch.float32, enforce_eager=True, max_model_len=160), cache_config=cc,
                      max_num_seqs=4, max_num_batched_tokens=chunk, async_scheduling=async_scheduling)
    model = build_model(arch, role="colocated", dtype=torch.float32, device="cpu", seed=0, max_positions=160)
    return LLMEngine(ec, model)


@pytest.mark.parametrize("preset", ["tiny-qwen3-moe", "tiny-dsv1", "tiny-qwen3.5"])
def test_prefill_and_decode_see_the_same_cache(preset):
    """A prompt in one piece, in chunks, or recomputed after preemption: the stored rows are the same,
    so the tokens are."""
    want = _engine(preset).generate(PROMPTS, 24)
    assert _engine(preset, chunk=16).generate(PROMPTS, 24) == want
    small = _engine(preset, num_blocks=13)
    assert small.generate(PROMPTS, 24) == want
    assert small.num_preemptions > 0
    assert _engine(preset, async_scheduling=True).generate(PROMPTS, 24) == want


def test_a_budget_that_is_never_reached_changes_nothing():
    want = _engine().generate(PROMPTS, 24)
    eng = _engine(kv_budget=120, kv_recent=16)
    assert eng.generate(PROMPTS, 24) == want and eng.num_evictions == 0
    assert eng.kv.scores.min() >= 0


def test_budget_bounds_the_cache():
    eng = _engine(kv_budget=32, kv_recent=8, kv_budget_slack=16)
    ids = [eng.add_request(p, 60) for p in PROMPTS]
    free0 = eng.kv.allocator.num_free
    first = eng.step()  # the prompts
    assert set(first) == set(ids)
    while eng.has_unfinished():
        eng.step()
        for r in eng.running:
            cached = r.num_tokens - 1 - r.evicted
            assert 0 <= cached <= 32 + 16
            # blocks for the next position at most, and never more than the bounded length needs
            assert len(r.blocks) <= -(-(32 + 16 + 1) // 16)
    assert eng.num_evictions >= 4
    assert [len(eng.finished[i].output) for i in ids] == [60] * 4
    assert eng.kv.allocator.num_free == free0  # every block came back
    assert sum(eng.kv.allocator._ref) == 0


def test_eviction_keeps_what_was_attended():
    """After a cut, each layer's cache holds the recent rows and the best scored of the others, in order."""
    eng = _engine(kv_budget=24, kv_recent=4, kv_budget_slack=8)
    eng.add_request(PROMPTS[0], 40)
    eng.step()
    r = eng.running[0]
    kv, scores = eng.kv.layer(0)
    assert isinstance(eng.kv.layer(0), Int4Layer)
    pos = torch.arange(37)
    blk, off = torch.tensor(r.blocks)[pos // 16], pos % 16
    w = scores[blk, :, off].t().clone()  # [kv_heads, 37]
    # every query of the prompt spreads a weight of 1 per head: 4 query heads on 2 KV heads
    torch.testing.assert_close(w.sum(1), torch.full((2,), 2.0 * 37), atol=1e-3, rtol=0)
    rows = kv.k[blk, :, off].clone()
    eng._keep_budget()
    assert r.evicted == 13 and eng.num_evictions == 1
    blk, off = torch.tensor(r.blocks)[torch.arange(24) // 16], torch.arange(24) % 16
    for h in range(2):
        keep = sorted(torch.topk(w[h, :33], 20).indices.tolist()) + [33, 34, 35, 36]
        assert torch.equal(kv.k[blk, h, off], rows[keep, h])
        torch.testing.assert_close(scores[blk, h, off], w[h, keep], rtol=0, atol=0)
    eng.step()  # decodes the next position behind the kept ones
    assert eng.running[0].num_tokens == 39


def test_int8_projections():
    plain = _engine(kv_cache_dtype="auto")
    quant = _engine(arch_kw={"attn_quant": "int8"}, kv_cache_dtype="auto")
    a, b = plain.model.layers[0].self_attn, quant.model.layers[0].self_attn
    assert b.qkv_proj.dtype == b.o_proj.dtype == torch.int8
    for w, q, s in ((a.qkv_proj, b.qkv_proj, b.qkv_scale), (a.o_proj, b.o_proj, b.o_scale)):
        half = w.abs().amax(1, keepdim=True) / 254 * (1 + 2.0**-16)
        assert ((q.float() * s[:, None] - w).abs() <= half).all()
    out = quant.generate(PROMPTS, 8)
    assert all(len(o) == 8 for o in out)
    both = _engine(arch_kw={"attn_quant": "int8"}, kv_budget=32, kv_recent=8, kv_budget_slack=4)
    assert all(len(o) == 40 for o in both.generate(PROMPTS, 40)) and both.num_evictions > 0


def test_refusals():
    for kw in (dict(kv_cache_dtype="fp8"), dict(kv_cache_dtype="auto", kv_budget=32), dict(kv_budget=0),
               dict(kv_budget=32, kv_recent=33), dict(kv_budget=32, kv_recent=-1), dict(kv_budget=32, kv_budget_slack=0),
               dict(kv_budget=32, kv_recent=8, enable_prefix_caching=True),
               dict(kv_budget=32, kv_recent=8, async_scheduling=True), dict(block_size=24)):
        with pytest.raises(ValueError):
            _engine(**kw)
    with pytest.raises(ValueError):
        _engine("tiny-dsv2")  # latent attention
    with pytest.raises(ValueError):
        _engine("tiny-qwen3-moe", arch_kw={"attn_quant": "int3"})
    with pytest.raises(ValueError):
        _engine("tiny-dsv2", arch_kw={"attn_quant": "int8"}, kv_cache_dtype="auto")
    eng = _engine()
    with pytest.raises(ValueError):
        eng.add_request([1, 2, 3], 4, hold_kv=True)
    with pytest.raises(ValueError):
        eng.add_prefilled_request(b"", 4)


def test_cache_sizes_and_synthetic_fill():
    arch = get_preset("tiny-qwen3-moe")
    bf16 = KVCache.bytes_per_block(arch, 64, torch.bfloat16)
    int4 = KVCache.bytes_per_block(arch, 64, torch.bfloat16, cache_dtype="int4")
    assert int4 * 16 / bf16 == 4.5
    scored = KVCache.bytes_per_block(arch, 64, torch.bfloat16, cache_dtype="int4", with_scores=True)
    L = len(arch.full_attention_layers)
    assert scored - int4 == L * 64 * arch.num_key_value_heads * 4
    cache = KVCache(arch, 4, 64, torch.bfloat16, "cpu", cache_dtype="int4")
    assert sum(t.numel() * t.element_size() for kv in cache.int4 for t in kv) == 4 * int4
    cache.fill_random_(seed=1)
    from afd_plugin_b200.ops import reference as ref

    v = ref.int4_dequantize(cache.int4[0].v, cache.int4[0].v_scale)
    assert abs(v.mean().item()) < 0.05 and 1.5 < v.std().item() < 2.5  # evenly spread over +- 3.3


def test_server_flags():
    from afd_plugin_b200.serving.__main__ import parse_args

    args = parse_args(["--kv-cache-dtype", "int4", "--kv-cache-budget", "512", "--attn-quant", "int8"])
    assert (args.kv_cache_dtype, args.kv_cache_budget, args.kv_cache_recent, args.attn_quant) == ("int4", 512, 128, "int8")
    args = parse_args([])
    assert (args.kv_cache_dtype, args.kv_cache_budget, args.attn_quant) == ("auto", None, None)
