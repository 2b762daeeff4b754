"""Bounded 4-bit cache under captured steps whose batch shrinks: padding rows touch no live sequence."""

import pytest
import torch

from afd_plugin_b200.engine_config import CacheConfig, CompilationConfig, EngineConfig, ModelConfig
from afd_plugin_b200.models import build_model, get_preset
from afd_plugin_b200.ops import _ext
from afd_plugin_b200.runtime.engine import LLMEngine

pytestmark = pytest.mark.gpu


def test_every_step_adds_the_weights_of_its_requests_only():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    bs = 16
    arch = get_preset("tiny-qwen3-moe")
    ec = EngineConfig(ModelConfig(arch, dtype=torch.bfloat16, max_model_len=256),
                      cache_config=CacheConfig(block_size=bs, kv_cache_dtype="int4", kv_budget=32, kv_recent=8,
                                               kv_budget_slack=4, num_blocks=24),
                      compilation_config=CompilationConfig(cudagraph_capture_sizes=[4]), max_num_seqs=4)
    eng = LLMEngine(ec, build_model(arch, role="colocated", dtype=torch.bfloat16, device="cuda", seed=0,
                                    max_positions=256))
    eng.capture_graphs()
    for i, n in enumerate((40, 29, 33, 30)):
        eng.add_request([(7 * i + j * j) % 250 for j in range(n)], 6 + 9 * i)  # they end one after another
    eng.step()
    group = arch.num_attention_heads // arch.num_key_value_heads
    cuts, padded = 0, 0
    while eng.running:
        cuts0 = eng.num_evictions
        eng._keep_budget()  # as the step does first; the step then finds nothing to cut
        cuts += eng.num_evictions - cuts0
        eng._reserve_decode_blocks()
        want = eng.kv.scores.clone()
        for r in eng.running:  # the rows this step writes start at zero
            place = r.num_tokens - 1 - r.evicted
            want[:, r.blocks[place // bs], :, place % bs] = 0
        n = len(eng.running)
        padded += n < 4
        live = sorted(b for r in eng.running for b in r.blocks)
        eng.step()
        added = (eng.kv.scores - want)[:, 1:]  # block 0 is the padding block
        # each of the n queries spreads a weight of 1 per query head over its own sequence
        torch.testing.assert_close(added.sum((1, 3)), torch.full_like(added[:, 0, :, 0], group * n), rtol=1e-4, atol=0)
        idle = torch.ones(added.shape[1], dtype=torch.bool)
        idle[torch.tensor(live) - 1] = False
        assert (added[:, idle.cuda()] == 0).all()
    assert cuts >= 6 and padded >= 10
    assert _ext.ops().read_status(0) == 0
