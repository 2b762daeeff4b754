"""The decode's own roundings against 64 bits: what is left beside the output's rounding to its type."""

import math

import pytest
import torch

from afd_plugin_b200 import ops
from afd_plugin_b200.ops import _ext

pytestmark = pytest.mark.gpu

# Of p * step in the second product: fp16 factors for bf16 results (half a step of 11 bits), two fp16 parts for fp16
# results (half a step of what the first leaves, 22 bits).
FACTOR = {torch.bfloat16: 2.0**-11, torch.float16: 2.0**-22}


def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    assert _ext.load(), "extension not built"


def check(q, kv, table, lens, scale, out):
    """Every result of ``out`` within the bound that the kernel's arithmetic gives; returns the largest share of it."""
    hkv, bs = kv.k.shape[1], kv.block_size
    heads, d = q.shape[1], q.shape[2]
    half = torch.finfo(q.dtype).eps / 2
    worst = 0.0
    for b, n in enumerate(lens):
        if n == 0:
            assert (out[b] == 0).all()
            continue
        pos = torch.arange(n, device=q.device)
        blk, off = table[b].long()[pos // bs], pos % bs

        def rows(codes, pairs):
            c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[blk, :, off].double() - 8
            step, zero = (pairs[blk, :, off].double()[..., i].repeat_interleave(64, -1) for i in (0, 1))
            return c, step, zero + 8 * step  # c * step + the last: the value

        ck, sk, zk = rows(kv.k, kv.k_scale)
        cv, sv, zv = rows(kv.v, kv.v_scale)
        qd = q[b].double().view(hkv, heads // hkv, d)
        s = torch.einsum("kgd,nkd->kgn", qd, ck * sk + zk) * scale
        p = torch.softmax(s, -1)
        want = torch.einsum("kgn,nkd->kgd", p, cv * sv + zv)
        # A logit is a sum of 64-dim sums and their scales in fp32: at most d / 16 + 8 roundings on its way, each
        # half a step (2^-24) of the terms' magnitude.  exp2 and the differences it takes add 2^-20.
        size = torch.einsum("kgd,nkd->kgn", qd.abs(), ck.abs() * sk + zk.abs()).amax(-1) * abs(scale)
        logit = (d / 16 + 8) * 2.0**-24 * size + 2.0**-20
        coded = torch.einsum("kgn,nkd->kgd", p, cv.abs() * sv)
        mag = coded + torch.einsum("kgn,nkd->kgd", p, zv.abs())
        # fp32 sums over the positions: at most one rounding per 16 of a warp's, and the merges
        sums = (n / 64 + 40) * 2.0**-24
        # factors far below the largest step of their sequence lose more: 2^-30 of it each
        tiny = 2.0**-30 * 8 * sv.amax((0, 2))[:, None, None] * n
        tol = (FACTOR[q.dtype] * coded + half * want.abs() + (2 * logit[..., None] + sums) * mag
               + tiny * p.amax(-1, keepdim=True) + torch.finfo(q.dtype).smallest_normal)
        share = ((out[b].double().view_as(want) - want).abs() / tol).max().item()
        assert share <= 1, (b, n, share)
        worst = max(worst, share)
    return worst


def _pool(lens, hkv, d, bs, seed):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // bs) for n in lens]
    ids = (torch.randperm(sum(need), generator=g) + 1).int().split(need)
    table = torch.zeros(len(lens), max(1, max(need)), dtype=torch.int32)
    for b, blocks in enumerate(ids):
        table[b, : len(blocks)] = blocks
    kv = ops.int4_kv_cache(sum(need) + 1, bs, hkv, d)
    slots = torch.arange(bs, (sum(need) + 1) * bs)
    k, v = (torch.randn(len(slots), hkv, d, generator=g) for _ in range(2))
    ops.gqa_cache_write_int4(kv, k.bfloat16().cuda(), v.bfloat16().cuda(), slots.cuda())
    return kv, table.cuda(), g


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,hkv,d,bs,lens", [
    (8, 1, 128, 64, [0, 1, 2, 15, 17, 40, 64]),      # one launch
    (16, 16, 128, 16, [700, 3, 129]),                # multi-head
    (64, 4, 128, 64, [1100, 17]),                    # 16 heads share the codes
    (16, 2, 256, 32, [0, 30, 530, 1025]),
    (24, 2, 64, 48, [900, 5, 100]),
    (7, 1, 64, 16, [40]),
    (32, 4, 128, 64, [9000, 1, 513]),
])
@pytest.mark.parametrize("spread", [0.3, 1.5, 12.0])  # flat and peaked probabilities
def test_results_are_within_their_own_rounding(heads, hkv, d, bs, lens, spread, dtype):
    _need_cuda()
    kv, table, g = _pool(lens, hkv, d, bs, heads + d)
    q = (spread * torch.randn(len(lens), heads, d, generator=g)).to(dtype).cuda()
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = ops.gqa_decode_int4(q, kv, table, lens_t, 1 / math.sqrt(d))
    check(q, kv, table, lens, 1 / math.sqrt(d), out)
    assert _ext.ops().read_status(0) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_value_steps_of_very_different_sizes(dtype):
    """Steps 2^12 apart: the power of two that holds a group's steps moves, the roundings stay."""
    _need_cuda()
    lens = [900, 40, 33]
    kv, table, g = _pool(lens, 1, 128, 64, 23)
    e = torch.randint(-6, 6, (*kv.v_scale.shape[:-1], 1), generator=g)
    kv.v_scale.copy_((kv.v_scale.float() * torch.exp2(e.float()).cuda()).bfloat16())
    q = torch.randn(3, 8, 128, generator=g).to(dtype).cuda()
    out = ops.gqa_decode_int4(q, kv, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), 0.1)
    check(q, kv, table, lens, 0.1, out)


def test_many_launches_with_scores():
    """More sequences than one launch takes, ragged, some empty: results, log-sum-exps and every score."""
    _need_cuda()
    g = torch.Generator().manual_seed(31)
    lens = [int(x) for x in torch.randint(0, 60, (600,), generator=g)]
    lens[255], lens[256], lens[511], lens[512] = 700, 0, 0, 777
    heads, hkv, d, bs = 6, 2, 64, 16
    kv, table, g = _pool(lens, hkv, d, bs, 32)
    q = torch.randn(600, heads, d, generator=g).bfloat16().cuda()
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    scores = torch.rand(kv.k.shape[:3], generator=g).cuda()
    before = scores.clone()
    out, lse = ops.gqa_decode_int4(q, kv, table, lens_t, 0.125, scores=scores, return_lse=True)
    check(q, kv, table, lens, 0.125, out)
    ks = ops.gqa_cache_read_int4(kv, torch.arange(kv.num_blocks * bs, device="cuda"), dtype=torch.float32)[0]
    want = before.double()
    for b, n in enumerate(lens):
        if n == 0:
            assert torch.isneginf(lse[b]).all()
            continue
        pos = torch.arange(n, device="cuda")
        blk, off = table[b].long()[pos // bs], pos % bs
        s = torch.einsum("kgd,nkd->kgn", q[b].double().view(hkv, -1, d), ks[blk * bs + off].double()) * 0.125
        ref = torch.logsumexp(s, -1)
        # logits below 64 in magnitude: their 16 roundings and those of the logarithm
        assert ((lse[b].double().view_as(ref) - ref).abs() <= 32 * 2.0**-24 * 64).all(), b
        want[blk, :, off] += torch.softmax(s, -1).sum(1).t()
    # three heads' weights, each off by a logit's error, added to a score below 4 (half a step: 2^-23)
    assert ((scores.double() - want).abs() <= 3 * 2 * 32 * 2.0**-24 * 64 + 2.0**-22).all()
    empty = torch.ones(kv.num_blocks, dtype=torch.bool)
    empty[table[torch.tensor(lens) > 0].cpu().unique().long()] = False
    assert torch.equal(scores[empty.cuda()], before[empty.cuda()])
