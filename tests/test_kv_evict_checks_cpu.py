"""Debug checks of the eviction: blocks that two sequences share are named before they are moved twice."""

import pytest
import torch

from afd_plugin_b200 import ops


@pytest.fixture
def checked():
    ops.checks.enable()
    yield
    ops.checks.enable(False)


def _evict(table, lens, budget):
    kv = ops.int4_kv_cache(9, 16, 1, 64, device="cpu")
    return ops.kv_evict_int4(kv, torch.zeros(9, 1, 16), torch.tensor(table, dtype=torch.int32),
                             torch.tensor(lens, dtype=torch.int32), budget, 1)


@pytest.mark.parametrize("table,lens", [
    ([[1, 2, 3], [4, 2, 0]], [40, 20]),   # two sequences that are cut
    ([[1, 2, 3], [3, 0, 0]], [40, 5]),    # one is not: its rows would be overwritten
    ([[5, 0, 0], [1, 5, 0]], [3, 20]),
    ([[1, 2, 1]], [40]),                  # twice in one sequence
])
def test_shared_blocks_are_named(checked, table, lens):
    with pytest.raises(ops.checks.KernelInputError, match="must not be shared"):
        _evict(table, lens, 10)


def test_blocks_that_nothing_moves_may_be_shared(checked):
    new, _ = _evict([[1, 2, 3], [1, 2, 0], [4, 5, 3]], [10, 9, 30], 16)  # entries past a length do not count
    assert new.tolist() == [10, 9, 16]
    _evict([[0, 0, 0], [0, 0, 0]], [0, 0], 1)
    new, _ = _evict([[1, 2, 0], [1, 2, 0]], [20, 20], 20)  # nothing is longer than the budget
    assert new.tolist() == [20, 20]
