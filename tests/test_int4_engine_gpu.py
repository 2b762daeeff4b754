"""The engine on the sm_100a kernels with the 4-bit KV cache, a cache budget and int8 projections."""

import pytest
import torch

from afd_plugin_b200.engine_config import CacheConfig, CompilationConfig, EngineConfig, ModelConfig
from afd_plugin_b200.models import build_model, get_preset
from afd_plugin_b200.ops import _ext
from afd_plugin_b200.runtime.engine import LLMEngine

pytestmark = pytest.mark.gpu

PROMPTS = [[(7 * i + j * j) % 250 for j in range(n)] for i, n in enumerate((90, 5, 33, 1))]


def _engine(preset="tiny-qwen3-moe", graphs=False, quant=None, **cache):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    arch = get_preset(preset).scaled(attn_quant=quant)
    ec = EngineConfig(ModelConfig(arch, dtype=torch.bfloat16, enforce_eager=not graphs, max_model_len=256),
                      cache_config=CacheConfig(**{"block_size": 32, "kv_cache_dtype": "int4", **cache}),
                      compilation_config=CompilationConfig(cudagraph_capture_sizes=[4]), max_num_seqs=4)
    eng = LLMEngine(ec, build_model(arch, role="colocated", dtype=torch.bfloat16, device="cuda", seed=0,
                                    max_positions=256))
    if graphs:
        eng.capture_graphs()
    return eng


@pytest.mark.parametrize("preset,quant", [("tiny-qwen3-moe", None), ("tiny-qwen3-moe", "int8"), ("tiny-dsv1", "int8"),
                                          ("tiny-qwen3.5", None)])
@pytest.mark.parametrize("budget", [None, 40])
def test_graphs_and_eager_steps_agree(preset, quant, budget):
    kw = {} if budget is None else {"kv_budget": budget, "kv_recent": 8, "kv_budget_slack": 8}
    eager, graphed = _engine(preset, False, quant, **kw), _engine(preset, True, quant, **kw)
    a, b = eager.generate(PROMPTS, 70), graphed.generate(PROMPTS, 70)
    assert a == b and all(len(o) == 70 for o in a)
    assert (eager.num_evictions > 0) == (budget is not None) and eager.num_evictions == graphed.num_evictions
    torch.cuda.synchronize()
    assert _ext.ops().read_status(0) == 0


def test_replayed_steps_read_the_moved_rows():
    """Between two replays of one captured step the cache is cut in place; the logits stay those of an
    engine that runs every step eagerly."""
    kw = {"kv_budget": 48, "kv_recent": 16, "kv_budget_slack": 4}
    eager, graphed = _engine(graphs=False, **kw), _engine(graphs=True, **kw)
    for e in (eager, graphed):
        for p in PROMPTS:
            e.add_request(p, 40)
    for _ in range(40):
        assert eager.step() == graphed.step()
        if eager.running:
            n = len(eager.running)
            assert torch.equal(eager.runner.last_logits[:n], graphed.runner.last_logits[:n])
    assert graphed.num_evictions >= 3
