"""Prefill attention sums its attention weights only where the cache keeps scores."""

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from afd_plugin_b200.engine_config import CacheConfig, EngineConfig, ModelConfig
from afd_plugin_b200.models import build_model, get_preset
from afd_plugin_b200.ops import reference as ref
from afd_plugin_b200.runtime.engine import LLMEngine


class _Reductions(TorchDispatchMode):
    """Sizes of the tensors that ``sum`` reduced."""

    def __init__(self):
        super().__init__()
        self.sizes = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.overloadpacket is torch.ops.aten.sum:
            self.sizes.append(args[0].dim())
        return func(*args, **(kwargs or {}))


def test_paged_prefill_reduces_nothing_it_does_not_return():
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn(3, 16, 2, 32, generator=g), torch.randn(3, 16, 2, 32, generator=g)
    q = torch.randn(7, 4, 32, generator=g)
    with _Reductions() as seen:
        ref.gqa_prefill(q, k, v, torch.tensor([2, 1], dtype=torch.int32), torch.arange(13, 20), 0.2)
    assert seen.sizes == []


@pytest.mark.parametrize("kv_budget", [None, 32])
def test_int4_prefill(kv_budget):
    arch = get_preset("tiny-qwen3-moe")
    ec = EngineConfig(ModelConfig(arch, dtype=torch.float32, enforce_eager=True, max_model_len=64),
                      cache_config=CacheConfig(block_size=16, kv_cache_dtype="int4", kv_budget=kv_budget, kv_recent=8),
                      max_num_seqs=2)
    eng = LLMEngine(ec, build_model(arch, role="colocated", dtype=torch.float32, seed=0, max_positions=64))
    eng.add_request(list(range(1, 20)), 4)
    with _Reductions() as seen:
        eng.step()
    # the weights are [tokens, kv heads, group, positions]
    assert seen.sizes.count(4) == (0 if kv_budget is None else len(arch.full_attention_layers))
