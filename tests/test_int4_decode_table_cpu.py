"""Under a cache budget the decode gets a block table of the bounded length, which always holds the sequences."""

import pytest
import torch

from afd_plugin_b200 import ops
from afd_plugin_b200.engine_config import CacheConfig, EngineConfig, ModelConfig
from afd_plugin_b200.models import build_model, get_preset
from afd_plugin_b200.runtime.engine import LLMEngine


def _engine(chunk=None, **cache):
    arch = get_preset("tiny-qwen3-moe")
    ec = EngineConfig(ModelConfig(arch, dtype=torch.float32, enforce_eager=True, max_model_len=160),
                      cache_config=CacheConfig(block_size=16, kv_cache_dtype="int4", **cache), max_num_seqs=4,
                      max_num_batched_tokens=chunk)
    return LLMEngine(ec, build_model(arch, role="colocated", dtype=torch.float32, seed=0, max_positions=160))


@pytest.fixture
def seen(monkeypatch):
    calls = []
    plain = ops.gqa_decode_int4

    def spy(q, kv, table, lens, scale, **kw):
        calls.append((table.shape[1], int(lens.max())))
        return plain(q, kv, table, lens, scale, **kw)

    monkeypatch.setattr(ops, "gqa_decode_int4", spy)
    return calls


@pytest.mark.parametrize("budget,recent,slack,blocks", [(32, 8, 16, 3), (33, 1, 1, 3), (16, 16, 1, 2), (20, 0, 30, 4)])
@pytest.mark.parametrize("chunk", [None, 16])
def test_bounded_table(seen, budget, recent, slack, blocks, chunk):
    eng = _engine(chunk, kv_budget=budget, kv_recent=recent, kv_budget_slack=slack)
    prompts = [[(7 * i + j * j) % 250 for j in range(n)] for i, n in enumerate((37, 5, 70, 1))]
    out = eng.generate(prompts, 60)
    assert all(len(o) == 60 for o in out) and eng.num_evictions >= 4
    assert {w for w, _ in seen} == {blocks}
    assert max(n for _, n in seen) == budget + slack  # the bound is reached, and never passed


def test_tables_without_a_budget_or_with_a_large_one(seen):
    _engine().generate([[1, 2, 3]], 3)
    _engine(kv_budget=150, kv_recent=8, kv_budget_slack=100).generate([[1, 2, 3]], 3)
    assert {w for w, _ in seen} == {10}


def test_device_resident_loops_refuse_a_budget():
    """They move every row on without a cut, past what the bounded table holds."""
    eng = _engine(kv_budget=32, kv_recent=8)
    with pytest.raises(ValueError, match="cache budget"):
        eng.runner.advance_on_device(1)
