"""Decode over the 4-bit cache at the ends of the number range: very large and very small rows and queries."""

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


@pytest.mark.parametrize("n,d,hkv,heads", [(50, 128, 2, 8), (900, 64, 1, 16), (700, 256, 2, 6)])
@pytest.mark.parametrize("qe,ke,ve", [
    (0, 0, 98), (0, 0, -98), (98, -98, 0), (-98, 98, 0), (60, -60, -60), (-60, 60, 60), (-98, 98, 98), (98, -98, -98),
    (110, -110, 0), (120, -120, -110),
])
def test_powers_of_two_change_nothing(qe, ke, ve, n, d, hkv, heads):
    """Queries, keys and values times powers of two give the 64-bit result of the same stored rows."""
    _need_cuda()
    bs = 64
    g = torch.Generator().manual_seed(n + d)
    k, v = (torch.randn(n, hkv, d, generator=g).bfloat16().float() for _ in range(2))
    q = torch.randn(1, heads, d, generator=g).bfloat16().float()
    kv = ops.int4_kv_cache(-(-n // bs) + 1, bs, hkv, d)
    slots = torch.arange(n, device="cuda") + bs
    ops.gqa_cache_write_int4(kv, k.cuda() * 2.0**ke, v.cuda() * 2.0**ve, slots)
    ks, vs = (x.double() for x in ops.gqa_cache_read_int4(kv, slots, dtype=torch.float32))
    table = torch.arange(1, -(-n // bs) + 1, dtype=torch.int32, device="cuda")[None]
    qs = (q.cuda() * 2.0**qe).bfloat16()
    scale = 1 / math.sqrt(d)
    out, lse = ops.gqa_decode_int4(qs, kv, table, torch.tensor([n], dtype=torch.int32, device="cuda"), scale,
                                   return_lse=True)
    qd = qs.double().view(hkv, heads // hkv, d)
    s = torch.einsum("kgd,nkd->kgn", qd, ks) * scale
    p = torch.softmax(s, -1)
    want = torch.einsum("kgn,nkd->kgd", p, vs)
    # A logit: d products of at most size |q| |k| in fp32, and 2^-16 for exp2, the sums and the logarithm.
    off = (d + 16) * 2.0**-23 * torch.einsum("kgd,nkd->kgn", qd.abs(), ks.abs()).amax(-1) * scale + 2.0**-16
    # p * step is rounded to fp16 (half a step: 2^-11 of at most 8 steps of p); a code's value is at most 2 max|v|
    # away from its group's middle, so 8 steps are below 2 max|v|.  Then the output's own bf16.
    top = vs.abs().amax((0, 2))[:, None, None]
    tol = 2.0**-11 * 2 * top + 2 * off[..., None] * top + 2.0**-8 * want.abs()
    got = out.double().view_as(want)
    assert got.isfinite().all()
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max().item()
    assert ((lse.double().view_as(off) - torch.logsumexp(s, -1)).abs() <= off + 2.0**-20).all()


def test_a_huge_step_after_tiny_ones():
    """Steps that span the whole range inside one sequence: the largest values decide, nothing overflows."""
    _need_cuda()
    n, d, bs = 640, 128, 64
    g = torch.Generator().manual_seed(8)
    v = torch.randn(n, 1, d, generator=g)
    e = torch.randint(-100, 99, (n, 1, 2), generator=g).repeat_interleave(64, -1)
    v = torch.ldexp(v, e)
    kv = ops.int4_kv_cache(n // bs + 1, bs, 1, d)
    slots = torch.arange(n, device="cuda") + bs
    ops.gqa_cache_write_int4(kv, torch.zeros(n, 1, d, device="cuda"), v.cuda(), slots)
    vs = ops.gqa_cache_read_int4(kv, slots, dtype=torch.float32)[1].double()
    table = torch.arange(1, n // bs + 1, dtype=torch.int32, device="cuda")[None]
    out = ops.gqa_decode_int4(torch.ones(1, 8, d, device="cuda", dtype=torch.bfloat16), kv, table,
                              torch.tensor([n], dtype=torch.int32, device="cuda"), 1.0)
    want = vs.mean(0)  # keys of zero: every position weighs the same
    # fp16's half step, 2^-11, of n terms (8 steps, below 2 max|v|) / n; then the output's own bf16
    tol = 2.0**-11 * 2 * vs.abs().amax((0, 1)) + 2.0**-8 * want.abs()
    assert out.isfinite().all() and ((out[0].double() - want).abs() <= tol).all()
