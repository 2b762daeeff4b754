"""Slots outside the 4-bit cache on CPU: skipped by the write, zeros from the read, as on the GPU."""

import torch

from afd_plugin_b200 import ops


def test_slots_outside_the_cache():
    g = torch.Generator().manual_seed(7)
    kv, scores = ops.int4_kv_cache(3, 16, 2, 64, device="cpu"), torch.ones(3, 2, 16)
    rows = torch.randn(5, 2, 64, generator=g)
    slots = torch.tensor([20, -1, 48, 3, -48])
    ops.gqa_cache_write_int4(kv, rows, -rows, slots, scores)
    good = ops.int4_kv_cache(3, 16, 2, 64, device="cpu")
    ops.gqa_cache_write_int4(good, rows[[0, 3]], -rows[[0, 3]], slots[[0, 3]])
    assert all(torch.equal(a, b) for a, b in zip(kv, good))  # nothing else was written
    assert (scores == 0).sum() == 4 and (scores[1, :, 4] == 0).all() and (scores[0, :, 3] == 0).all()
    for back, x in zip(ops.gqa_cache_read_int4(kv, slots, dtype=torch.float32), (rows, -rows)):
        assert (back[[1, 2, 4]] == 0).all()
        assert (back[[0, 3]] - x[[0, 3]]).abs().max() < 0.4  # half a step of about 0.3
    empty = ops.gqa_cache_read_int4(kv, slots[:0])
    assert empty[0].shape == (0, 2, 64)
