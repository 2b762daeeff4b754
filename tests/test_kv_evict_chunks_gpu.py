"""Eviction whose move takes many chunks per CTA, while another stream keeps the memory busy: bit for bit."""

import math

import pytest
import torch

from afd_plugin_b200 import ops
from afd_plugin_b200.ops import _ext

pytestmark = pytest.mark.gpu


def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    assert _ext.load(), "extension not built"


def _plain(tensors, table, lens, budget, recent):
    """Positions kept, and the cache tensors ``[blocks, heads, block, ...]`` after the move (by whole rows)."""
    scores = tensors[-1]
    hkv, bs = scores.shape[1], scores.shape[2]
    out = [t.clone() for t in tensors]
    kept = torch.full((len(lens), hkv, budget), -1, dtype=torch.int32, device="cuda")
    heads = torch.arange(hkv, device="cuda")[:, None]
    for b, n in enumerate(lens):
        pos = torch.arange(n, device="cuda")
        if n <= budget:
            kept[b, :, :n] = pos.int()
            continue
        blk, off = table[b].long()[pos // bs], pos % bs
        w = scores[blk, :, off].t()[:, : n - recent]
        best = torch.sort(w, dim=-1, descending=True, stable=True).indices[:, : budget - recent]
        keep = torch.cat([best, pos[n - recent :].expand(hkv, -1)], 1).sort(-1).values
        kept[b] = keep.int()
        for t, o in zip(tensors, out):
            o[blk[:budget], heads, off[:budget]] = t[blk[keep], heads, off[keep]]
    return out, kept


@pytest.mark.parametrize("lens,hkv,dim,bs,budget,recent", [
    # a chunk is 512, 256 or 128 rows (dim 64, 128, 256) for each CTA of the cluster
    ([20011], 2, 64, 64, 18001, 100),             # eight CTAs: five chunks of 4096
    ([20011], 2, 128, 64, 19001, 1),              # ten of 2048
    ([9000, 12000], 1, 256, 48, 8999, 0),         # nine of 1024
    ([4000 + 7 * i for i in range(40)], 4, 128, 16, 3333, 64),   # one CTA: fourteen of 256
    ([3000 + 11 * i for i in range(40)], 4, 256, 16, 2500, 64),  # twenty of 128
    ([3500 + 11 * i for i in range(40)], 4, 64, 64, 3100, 5),    # seven of 512
], ids=lambda x: str(x if isinstance(x, int) else f"n{len(x)}x{x[0]}"))
def test_many_chunks_beside_a_busy_stream(lens, hkv, dim, bs, budget, recent):
    _need_cuda()
    g = torch.Generator(device="cuda")
    g.manual_seed(dim + len(lens))
    need = [math.ceil(n / bs) for n in lens]
    total = sum(need) + 1
    ids = (torch.randperm(total - 1, generator=g, device="cuda") + 1).int().cpu().split(need)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32)
    for b, blocks in enumerate(ids):
        table[b, : len(blocks)] = blocks
    table = table.cuda()
    kv = ops.int4_kv_cache(total, bs, hkv, dim)
    for t in (kv.k, kv.v):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, device="cuda", dtype=torch.uint8))
    for t in (kv.k_scale, kv.v_scale):
        t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
    scores = (torch.rand(kv.k.shape[:3], generator=g, device="cuda") * 1000).floor()  # ties among them
    start = [t.clone() for t in (*kv, scores)]
    want, want_kept = _plain(start, table, lens, budget, recent)
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    busy = torch.cuda.Stream()
    a, b = (torch.zeros(1 << 28, dtype=torch.uint8, device="cuda") for _ in range(2))
    for _ in range(6):
        for t, s in zip((*kv, scores), start):
            t.copy_(s)
        busy.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(busy):
            for _ in range(8):
                b.copy_(a)
        new, kept = ops.kv_evict_int4(kv, scores, table, lens_t, budget, recent)
        torch.cuda.synchronize()
        assert new.tolist() == [min(n, budget) for n in lens]
        assert torch.equal(kept, want_kept)
        for t, w in zip((*kv, scores), want):
            assert torch.equal(t, w)
    assert _ext.ops().read_status(0) == 0
