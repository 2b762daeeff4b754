"""Staged block-table rows when a request's blocks change in another way than by growing."""

from __future__ import annotations

import torch

from afd_plugin_b200.engine_config import CacheConfig, EngineConfig, ModelConfig
from afd_plugin_b200.models import build_model, get_preset
from afd_plugin_b200.runtime.engine import LLMEngine
from afd_plugin_b200.runtime.kv_cache import PAD_BLOCK


def _engine(preset, **cache):
    arch = get_preset(preset)
    ec = EngineConfig(ModelConfig(arch, dtype=torch.float32, enforce_eager=True, max_model_len=64),
                      cache_config=CacheConfig(**cache), max_num_seqs=4)
    return LLMEngine(ec, build_model(arch, role="colocated", dtype=torch.float32, seed=0, max_positions=64))


def _staged(eng, run_b):
    eng._stage_decode_inputs(eng.running, run_b)
    return eng._n_table[:run_b].tolist()


def _rows(eng, run_b):
    rows = [r.blocks + [PAD_BLOCK] * (eng.max_blocks_per_seq - len(r.blocks)) for r in eng.running]
    return rows + [[PAD_BLOCK] * eng.max_blocks_per_seq] * (run_b - len(rows))


def test_a_recomputed_request_comes_back_to_its_row_with_other_blocks():
    eng = _engine("tiny-dsv2", block_size=4)
    for n in (5, 9, 6):
        eng.add_request(list(range(1, n + 1)), 20)
    eng.step()
    assert _staged(eng, 3) == _rows(eng, 3)
    last = eng.running.pop()
    old = list(last.blocks)
    eng._preempt(last)
    eng.kv.allocator.allocate(1)  # another sequence grows meanwhile
    eng.step()  # recomputed: the same row, as many blocks as before
    assert eng.running[2] is last and len(last.blocks) == len(old) and last.blocks != old
    assert _staged(eng, 3) == _rows(eng, 3)


def test_padding_rows_hold_no_blocks_after_a_cut():
    """One request ends on the step before another is cut to the budget: its row turns into padding."""
    eng = _engine("tiny-qwen3-moe", block_size=16, kv_cache_dtype="int4", kv_budget=20, kv_recent=4, kv_budget_slack=8)
    for n, out in ((20, 40), (9, 9)):
        eng.add_request(list(range(1, n + 1)), out)
    eng.step()
    assert _staged(eng, 4) == _rows(eng, 4)
    while eng.num_evictions == 0:
        ended = len(eng.running) == 1
        eng.step()
    assert ended and len(eng.running) == 1 and len(eng.finished) == 1
    assert _staged(eng, 4) == _rows(eng, 4)


def test_a_cut_request_keeps_its_row():
    """A cut gives blocks back and the sequence grows again, to a block count it had with other blocks."""
    eng = _engine("tiny-qwen3-moe", block_size=16, kv_cache_dtype="int4", kv_budget=16, kv_recent=4, kv_budget_slack=20)
    for n in (20, 30):
        eng.add_request(list(range(1, n + 1)), 30)
    eng.step()
    changed = False
    seen = {}
    while eng.running:
        assert _staged(eng, 3) == _rows(eng, 3)
        for r in eng.running:
            old = seen.setdefault((r.req_id, len(r.blocks)), list(r.blocks))
            changed |= old != r.blocks
        eng.step()
        if eng.num_evictions and eng.kv.allocator.num_free > 3:
            eng.kv.allocator.allocate(1)  # others grow meanwhile
    assert changed
