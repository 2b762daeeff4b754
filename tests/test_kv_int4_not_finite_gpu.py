"""Rows that are not finite through the sm_100a cache write, read and decode: NaN stays NaN, where it was."""

import math

import pytest
import torch

from afd_plugin_b200 import ops
from afd_plugin_b200.ops import _ext

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan


def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    assert _ext.load(), "extension not built"


def _spoilt(tokens, hkv, d, dtype, seed):
    """Random rows, and which (token, head, group) hold something that is not finite."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, hkv, d, generator=g)
    spoilt = torch.zeros(tokens, hkv, d // 64, dtype=torch.bool)
    for t in range(0, tokens, 2):
        for h in range(hkv):
            j = int(torch.randint(0, d // 64, (1,), generator=g))
            spoilt[t, h, j] = True
            group = x[t, h, 64 * j : 64 * j + 64]
            at = torch.randperm(64, generator=g)
            kind = (t // 2 + h) % 7
            if kind < 3:
                group[at[0]] = (NAN, INF, -INF)[kind]
            elif kind == 3:
                group[at[:3]] = torch.tensor([INF, NAN, -INF])
            else:
                group[:] = (INF, -INF, NAN)[kind - 4]
    return x.to(dtype), spoilt


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hkv,d,bs", [(1, 64, 16), (3, 128, 32), (2, 256, 64)])
def test_write_and_read(hkv, d, bs, dtype):
    _need_cuda()
    tokens = 61
    k, bad_k = _spoilt(tokens, hkv, d, dtype, 1)
    v, bad_v = _spoilt(tokens, hkv, d, dtype, 2)
    kv, cpu = ops.int4_kv_cache(4, bs, hkv, d), ops.int4_kv_cache(4, bs, hkv, d, device="cpu")
    slots = torch.randperm(4 * bs, generator=torch.Generator().manual_seed(3))[: min(tokens, 4 * bs)]
    n = len(slots)
    ops.gqa_cache_write_int4(kv, k[:n].cuda(), v[:n].cuda(), slots.cuda())
    ops.gqa_cache_write_int4(cpu, k[:n], v[:n], slots)
    for a, b in zip(kv, cpu):  # the same bits, NaN pairs included
        assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))
    for dt in (torch.float32, dtype):
        for back, x, bad in zip(ops.gqa_cache_read_int4(kv, slots.cuda(), dtype=dt), (k, v), (bad_k, bad_v)):
            nan = back.isnan().cpu().unflatten(-1, (-1, 64))
            assert nan[bad[:n]].all() and not nan[~bad[:n]].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,bs", [(50, 16), (900, 64)])  # one launch, and shares over CTAs
def test_decode_over_a_spoilt_position(n, bs, dtype):
    """A key group that is not finite spoils its head's results whole; a value group its own dims."""
    _need_cuda()
    d, hkv, heads = 128, 4, 8
    g = torch.Generator().manual_seed(4)
    k, v = torch.randn(n, hkv, d, generator=g), torch.randn(n, hkv, d, generator=g)
    k[n // 2, 1, 70], k[n - 1, 2, 3] = NAN, INF
    v[n // 3, 3, 100] = NAN
    kv = ops.int4_kv_cache(n // bs + 2, bs, hkv, d)
    slots = torch.arange(n) + bs
    ops.gqa_cache_write_int4(kv, k.cuda(), v.cuda(), slots.cuda())
    table = (torch.arange(n // bs + 1, dtype=torch.int32) + 1)[None]
    q = torch.randn(1, heads, d, generator=g).to(dtype)
    scores = torch.zeros(kv.k.shape[:3], device="cuda")
    out, lse = ops.gqa_decode_int4(q.cuda(), kv, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), 0.1,
                                   scores=scores, return_lse=True)
    nan = out.isnan().cpu().view(hkv, heads // hkv, d)
    want = torch.zeros_like(nan)
    want[1:3] = True
    want[3, :, 64:] = True
    assert torch.equal(nan, want)
    assert torch.equal(lse.isnan().cpu().view(hkv, -1), want[:, :, 0])
    w = scores[1 + torch.arange(n) // bs, :, torch.arange(n) % bs].cpu()
    assert w[:, 1:3].isnan().all() and w[:, [0, 3]].isfinite().all()
