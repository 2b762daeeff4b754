"""The 4-bit KV cache on CPU: the definitions against exact arithmetic, the entry points' refusals."""

import math
from fractions import Fraction

import pytest
import torch

from afd_plugin_b200 import ops
from afd_plugin_b200.ops import reference as ref


def _bf16_neighbours(x: float):
    """The bf16 values at or below / at or above ``x`` (by a walk over the encoding)."""
    t = torch.tensor(x, dtype=torch.float64).to(torch.bfloat16)
    lo = hi = t
    while lo.double().item() > x:
        lo = torch.nextafter(lo, torch.tensor(-math.inf, dtype=torch.bfloat16))
    while hi.double().item() < x:
        hi = torch.nextafter(hi, torch.tensor(math.inf, dtype=torch.bfloat16))
    return lo.double().item(), hi.double().item()


def _f32(x: Fraction) -> float:
    """Rounded to the nearest fp32 value, ties to even, by exact comparison."""
    t = torch.tensor(float(x), dtype=torch.float64).to(torch.float32)
    best = [torch.nextafter(t, torch.tensor(s * math.inf)) for s in (-1, 1)] + [t]
    near = min(abs(Fraction(b.item()) - x) for b in best)
    tied = [b for b in best if abs(Fraction(b.item()) - x) == near]
    return next(b for b in tied if len(tied) == 1 or b.view(torch.int32).item() % 2 == 0).item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_definition(dtype):
    g = torch.Generator().manual_seed(3)
    rows = (torch.randn(6, 64, generator=g) * torch.tensor([1, 1e-3, 40, 1, 1e-20, 7])[:, None]).to(dtype)
    rows[3] = 2.5  # constant: no step
    rows[5] = rows[5].abs() + 3  # a positive minimum
    codes, scale = ref.int4_quantize(rows)
    vals = ref.int4_dequantize(codes, scale)
    for x, c, (step, zero), v in zip(rows, torch.stack([codes & 15, codes >> 4], -1).flatten(-2), scale[:, 0], vals):
        xs = [Fraction(t) for t in x.double().tolist()]
        want_zero = _bf16_neighbours(float(min(xs)))[0]
        assert zero.item() == want_zero
        span = _f32(max(xs) - Fraction(want_zero))
        want_step = _bf16_neighbours(_f32(Fraction(span) / 15))[1]
        assert step.item() == want_step
        for xi, ci, vi in zip(xs, c.tolist(), v.tolist()):
            want = 0
            if want_step > 0:
                quot = _f32(Fraction(_f32(xi - Fraction(want_zero))) / Fraction(want_step))
                want = min(max(round(Fraction(quot)), 0), 15)  # round() of a Fraction takes ties to even
            assert ci == want
            assert vi == _f32(Fraction(want_zero) + want * Fraction(want_step))
            assert abs(vi - float(xi)) <= want_step / 2 * (1 + 2.0**-18) + abs(float(xi)) * 2.0**-22


def test_write_read_decode_and_scores_plain():
    g = torch.Generator().manual_seed(4)
    kv = ops.int4_kv_cache(6, 16, 2, 64, device="cpu")
    n, heads = 37, 6
    table = torch.tensor([[3, 1, 5], [0, 0, 0]], dtype=torch.int32)
    pos = torch.arange(n)
    slots = table[0].long()[pos // 16] * 16 + pos % 16
    k, v = torch.randn(n, 2, 64, generator=g), torch.randn(n, 2, 64, generator=g)
    scores = torch.full((6, 2, 16), 5.0)
    ops.gqa_cache_write_int4(kv, k, v, slots, scores)
    assert (scores[3] == 0).all() and (scores[2] == 5).all()
    rk, rv = ops.gqa_cache_read_int4(kv, slots, dtype=torch.float32)
    q = torch.randn(2, heads, 64, generator=g)
    lens = torch.tensor([n, 0], dtype=torch.int32)
    out, lse = ops.gqa_decode_int4(q, kv, table, lens, 0.2, scores=scores, return_lse=True)
    for h in range(heads):
        s = [(q[0, h].double() @ rk[t, h // 3].double()).item() * 0.2 for t in range(n)]
        top = max(s)
        z = sum(math.exp(x - top) for x in s)
        assert abs(lse[0, h].item() - top - math.log(z)) < 1e-5
        o = sum(math.exp(x - top) / z * rv[t, h // 3].double() for t, x in enumerate(s))
        torch.testing.assert_close(out[0, h].double(), o, atol=1e-5, rtol=0)
    assert (out[1] == 0).all() and torch.isneginf(lse[1]).all()
    # three heads share each KV head: their weights sum to 3 over the sequence
    for h in range(2):
        w = scores[:, h].flatten()[slots]
        assert abs(w.sum().item() - 3) < 1e-5
    assert (scores[2] == 5).all()


def test_refusals():
    kv = ops.int4_kv_cache(4, 16, 2, 64, device="cpu")
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.tensor([3, 4], dtype=torch.int32)
    q = torch.randn(2, 4, 64)
    ok = lambda **kw: ops.gqa_decode_int4(**{**dict(q=q, kv=kv, block_table=table, seq_lens=lens, scale=1.0), **kw})  # noqa: E731
    ok()
    for kw in (dict(q=q[..., :32]), dict(q=q[:, :3]), dict(q=q[:1]), dict(seq_lens=lens.long()),
               dict(block_table=table.long()), dict(block_table=table[:1]), dict(scores=torch.zeros(3, 2, 16)),
               dict(scores=torch.zeros(4, 2, 16).double()), dict(kv=ops.Int4KV(kv.k.int(), *kv[1:])),
               dict(kv=ops.Int4KV(kv.k, kv.k_scale.float(), kv.v, kv.v_scale)),
               dict(kv=ops.Int4KV(*(t[:, :, :8] for t in kv))), dict(kv=ops.Int4KV(*(t[:, :, ::2] for t in kv)))):
        with pytest.raises(ValueError):
            ok(**kw)
    k, slots = torch.randn(3, 2, 64), torch.arange(3)
    for a in ((k[:, :1], k, slots), (k, k.half(), slots), (k, k[:2], slots), (k, k, slots.int()), (k, k, slots[:2]),
              (k.double(), k.double(), slots)):
        with pytest.raises(ValueError):
            ops.gqa_cache_write_int4(kv, *a)
    with pytest.raises(ValueError):
        ops.gqa_cache_read_int4(kv, slots.int())
    for bad in (dict(head_dim=96), dict(block_size=24), dict(block_size=0)):
        with pytest.raises(ValueError):
            ops.int4_kv_cache(**{**dict(num_blocks=2, block_size=64, kv_heads=1, head_dim=64, device="cpu"), **bad})


def test_debug_checks_name_the_bad_entry():
    kv = ops.int4_kv_cache(4, 16, 1, 64, device="cpu")
    k = torch.randn(2, 1, 64)
    ops.checks.enable()
    try:
        with pytest.raises(ops.checks.KernelInputError):
            ops.gqa_cache_write_int4(kv, k, k, torch.tensor([0, 64]))
        with pytest.raises(ops.checks.KernelInputError):
            ops.gqa_decode_int4(torch.randn(1, 1, 64), kv, torch.tensor([[4]], dtype=torch.int32),
                                torch.tensor([3], dtype=torch.int32), 1.0)
    finally:
        ops.checks.enable(False)


@pytest.mark.parametrize("recent", [0, 3, 8])
def test_evict_keeps_the_best_and_the_recent(recent):
    g = torch.Generator().manual_seed(recent)
    bs, budget, lens = 16, 8, [37, 8, 0, 20]
    kv = ops.int4_kv_cache(9, bs, 2, 64, device="cpu")
    for t in (kv.k, kv.v):
        t.copy_(torch.randint(0, 256, t.shape, generator=g))
    for t in (kv.k_scale, kv.v_scale):
        t.copy_(torch.randn(t.shape, generator=g))
    scores = torch.randint(0, 4, kv.k.shape[:3], generator=g).float()  # ties
    scores[1, 0, 2], scores[1, 0, 3] = float("nan"), float("inf")
    table = torch.tensor([[1, 4, 2], [5, 0, 0], [0, 0, 0], [7, 3, 0]], dtype=torch.int32)
    old = [t.clone() for t in (*kv, scores)]
    new, kept = ops.kv_evict_int4(kv, scores, table, torch.tensor(lens, dtype=torch.int32), budget, recent)
    assert new.tolist() == [8, 8, 0, 8]
    at = lambda b, i: (int(table[b, i // bs]), i % bs)  # noqa: E731
    for b, n in enumerate(lens):
        for h in range(2):
            keep = list(range(n))
            if n > budget:
                w = [old[4][at(b, i)[0], h, at(b, i)[1]].item() for i in range(n - recent)]
                rank = sorted(range(n - recent), key=lambda i: (-(w[i] if w[i] == w[i] else -math.inf), i))
                keep = sorted(rank[: budget - recent]) + list(range(n - recent, n))
            assert kept[b, h].tolist() == keep + [-1] * (budget - len(keep))
            for i in range(n):  # kept rows first, the rest as they were
                src = at(b, keep[i] if i < len(keep) else i)
                for t, o in zip((*kv, scores), old):
                    torch.testing.assert_close(t[at(b, i)[0], h, at(b, i)[1]], o[src[0], h, src[1]], rtol=0, atol=0,
                                               equal_nan=True)
    for a in ((0, 0), (4, 5), (4, -1)):
        with pytest.raises(ValueError):
            ops.kv_evict_int4(kv, scores, table, torch.tensor(lens, dtype=torch.int32), *a)


def test_evict_refuses_positions_past_2_30():
    kv = ops.int4_kv_cache(2, 16, 1, 64, device="cpu")
    scores, lens = torch.zeros(2, 1, 16), torch.zeros(1, dtype=torch.int32)
    wide = torch.zeros(1, 1, dtype=torch.int32).expand(1, 2**26 + 1)
    with pytest.raises(ValueError, match="2\\^30"):
        ops.kv_evict_int4(kv, scores, wide, lens, 4, 1)
    for budget, recent in ((2**30 + 1, 0), (2**31, 1)):
        with pytest.raises(ValueError, match="2\\^30"):
            ops.kv_evict_int4(kv, scores, wide[:, :2], lens, budget, recent)
