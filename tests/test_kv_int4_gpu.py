"""sm_100a kernels of the 4-bit KV cache against 64-bit restatements."""

import math

import pytest
import torch

from afd_plugin_b200 import ops
from afd_plugin_b200.ops import _ext

pytestmark = pytest.mark.gpu

GROUP = 64


def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    assert _ext.load(), "extension not built"


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _codes64(codes, scale):
    """(c - 8, step, zero) of packed rows [..., d / 2], as fp64 [..., d]."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    step, zero = (scale.double()[..., i].repeat_interleave(GROUP, -1) for i in (0, 1))
    return c - 8, step, zero


def _pool(lens, hkv, d, bs, g, extra_blocks=3, width=None):
    """Random cache with shuffled blocks; everything no sequence reaches holds NaN scales and random codes."""
    need = [-(-n // bs) for n in lens]
    total = sum(need) + extra_blocks
    width = width or max(1, max(need))
    ids = (torch.randperm(total - 1, generator=g, device="cuda") + 1).tolist()
    table = torch.full((len(lens), width), 0, dtype=torch.int32)
    kv = ops.int4_kv_cache(total, bs, hkv, d)
    for t in (kv.k, kv.v):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, device="cuda", dtype=torch.uint8))
    for t in (kv.k_scale, kv.v_scale):
        t.fill_(float("nan"))
    at = 0
    for b, n in enumerate(lens):
        blocks = ids[at : at + need[b]]
        at += need[b]
        table[b, : len(blocks)] = torch.tensor(blocks, dtype=torch.int32)
        if n:
            pos = torch.arange(n, device="cuda")
            blk, off = table[b].cuda().long()[pos // bs], pos % bs
            for t in (kv.k_scale, kv.v_scale):
                step = 0.05 + torch.rand(n, hkv, d // GROUP, generator=g, device="cuda")
                zero = -7 * step + torch.randn(n, hkv, d // GROUP, generator=g, device="cuda")
                t[blk, :, off] = torch.stack([step, zero], -1).bfloat16()
    return kv, table.cuda()


def _gather(codes, scale, row, n, bs):
    pos = torch.arange(n, device=codes.device)
    blk, off = row.long()[pos // bs], pos % bs
    return _codes64(codes[blk, :, off], scale[blk, :, off])  # [n, hkv, d] each


def _check_decode(q, kv, table, lens, scale, out, lse, added=None):
    hkv, bs = kv.k.shape[1], kv.block_size
    heads, d = q.shape[1], q.shape[2]
    half = torch.finfo(q.dtype).eps / 2
    if added is not None:
        left = added.clone()
    for b, n in enumerate(lens):
        if n == 0:
            assert (out[b] == 0).all() and torch.isneginf(lse[b]).all()
            continue
        ck, sk, zk = _gather(kv.k, kv.k_scale, table[b], n, bs)
        cv, sv, zv = _gather(kv.v, kv.v_scale, table[b], n, bs)
        qd = q[b].double().view(hkv, heads // hkv, d)
        s = torch.einsum("kgd,nkd->kgn", qd, zk + (ck + 8) * sk) * scale
        p = torch.softmax(s, -1)
        want = torch.einsum("kgn,nkd->kgd", p, zv + (cv + 8) * sv)
        # a logit: d products and the group sums, each fp32 step of the magnitude of the terms
        size = torch.einsum("kgd,nkd->kgn", qd.abs(), ck.abs() * sk + (zk + 8 * sk).abs()).amax(-1) * scale
        off = (d + 16) * 2.0**-23 * size + 2.0**-16  # and exp2, the sums of the probabilities, the logarithm
        mag = torch.einsum("kgn,nkd->kgd", p, cv.abs() * sv + (zv + 8 * sv).abs())
        # p * step is rounded to bf16 (half a step: 2^-8), the output to its type
        tol = (2.0**-8 * torch.einsum("kgn,nkd->kgd", p, cv.abs() * sv) + half * want.abs()
               + 2 * off[..., None] * mag + torch.finfo(q.dtype).smallest_normal)
        err = (out[b].double().view_as(want) - want).abs()
        assert (err <= tol).all(), (b, n, (err / tol).max().item())
        ref_lse = torch.logsumexp(s, -1).flatten()
        assert ((lse[b].double() - ref_lse).abs() <= off.flatten() + 2.0**-22 * ref_lse.abs()).all(), (b, n)
        if added is not None:
            pos = torch.arange(n, device=q.device)
            blk, o = table[b].long()[pos // bs], pos % bs
            got = added[blk, :, o].double().t()  # [hkv, n]
            w = p.sum(1)
            # the weight's own error, and half a step of the fp32 score it was added to (below 2)
            assert ((got - w).abs() <= (p * 2 * off[..., None]).sum(1) + 2.0**-23).all(), (b, n)
            left[blk, :, o] = 0
    if added is not None:
        assert (left == 0).all(), "scores changed outside the sequences"


CASES = [
    # heads, kv_heads, dim, block, lens, table width in blocks (None: the longest)
    (8, 1, 128, 64, [0, 1, 15, 16, 17, 63, 64, 65], None),
    (32, 4, 128, 64, [512, 1, 0, 333], None),                 # one launch: at most 512 positions
    (32, 4, 128, 64, [1, 513, 0, 2000, 64, 1999], None),      # shares over CTAs
    (16, 16, 128, 16, [700, 3, 129], None),                   # multi-head, small blocks
    (16, 2, 256, 32, [0, 1, 530, 1025, 48], None),
    (64, 4, 128, 64, [1100, 17, 0], None),                    # 16 heads per KV head
    (28, 4, 128, 64, [600, 31], None),                        # 7
    (24, 2, 64, 48, [900, 5, 0, 100], None),                  # 12, dim 64
    (5, 1, 64, 16, [40], None),
    (40, 1, 128, 64, [777, 40], None),                        # 40: three passes of 16
    (20, 1, 256, 64, [700, 0, 9], None),                      # 20 at dim 256: three passes of 8
    (8, 2, 128, 64, [0, 0, 0], 20),                           # nothing anywhere
    (8, 1, 128, 64, [20000], None),                           # one sequence over every CTA
    (8, 2, 128, 64, [5, 9], 100),                             # short sequences, wide table
    (4, 2, 64, 64, [1] * 2100, 9),                            # more sequences than one launch takes
    (64, 4, 128, 64, [700, 0, 1500], 16500),                  # a table too wide for stored logits: scores from K again
    (6, 2, 64, 16, [900, 33, 1], 260000),
    (8, 1, 256, 64, [100, 700], 65536),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"h{c[0]}-{c[1]}-d{c[2]}-bs{c[3]}-n{len(c[4])}x{max(c[4])}")
def test_decode(case, dtype):
    _need_cuda()
    heads, hkv, d, bs, lens, width = case
    g = _gen(heads * 1000 + d)
    kv, table = _pool(lens, hkv, d, bs, g, width=width)
    q = torch.randn(len(lens), heads, d, generator=g, device="cuda").to(dtype)
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    scale = 1 / math.sqrt(d)
    out, lse = ops.gqa_decode_int4(q, kv, table, lens_t, scale, return_lse=True)
    scores = torch.rand(kv.k.shape[:3], generator=g, device="cuda")
    before = scores.clone()
    out2 = ops.gqa_decode_int4(q, kv, table, lens_t, scale, scores=scores)
    assert torch.equal(out, out2)
    if len(lens) > 100:
        lens, keep = lens[:6], [0, 1, 511, 512, 2047, 2099]
        q, table, out, lse = (t[keep] for t in (q, table, out, lse))
        _check_decode(q, kv, table, lens, scale, out, lse)
        return
    # what was added, with the score's own rounding counted in the tolerance
    _check_decode(q, kv, table, lens, scale, out, lse, scores.double() - before.double())
    assert _ext.ops().read_status(0) == 0


def test_decode_strided_query_and_table():
    _need_cuda()
    g = _gen(5)
    lens = [70, 600, 33]
    kv, table = _pool(lens, 2, 128, 64, g)
    wide = torch.randn(3, 16, 3, 200, generator=g, device="cuda").bfloat16()
    q = wide[:, :, 1, 7:135]  # odd start, strides that are not a row
    big = torch.zeros(3, table.shape[1] + 5, dtype=torch.int32, device="cuda")
    big[:, : table.shape[1]] = table
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = ops.gqa_decode_int4(q, kv, big[:, : table.shape[1]], lens_t, 0.1, return_lse=True)
    _check_decode(q, kv, table, lens, 0.1, out, lse)


def test_decode_large_logits():
    """Logits in the thousands: one position takes all the weight, early or late in the sequence."""
    _need_cuda()
    g = _gen(6)
    lens = [900, 17, 520]
    kv, table = _pool(lens, 2, 128, 64, g)
    q = 100 * torch.randn(3, 16, 128, generator=g, device="cuda").bfloat16()
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = ops.gqa_decode_int4(q, kv, table, lens_t, 1.0, return_lse=True)
    _check_decode(q, kv, table, lens, 1.0, out, lse)


def test_decode_lengths_and_blocks_out_of_range():
    """Negative and overlong lengths are clamped to the table; a bad block id is reported, not followed."""
    _need_cuda()
    g = _gen(7)
    kv, table = _pool([64, 64], 1, 64, 64, g)
    q = torch.randn(2, 4, 64, generator=g, device="cuda").bfloat16()
    lens = torch.tensor([-5, 1000], dtype=torch.int32, device="cuda")
    out, lse = ops.gqa_decode_int4(q, kv, table, lens, 0.1, return_lse=True)
    _check_decode(q, kv, table, [0, 64], 0.1, out, lse)
    C = _ext.ops()
    assert C.read_status(0) == 0
    table[1, 0] = 10_000_000
    try:
        ops.gqa_decode_int4(q, kv, table, lens, 0.1)
        torch.cuda.synchronize()
        assert C.read_status(0) != 0
    finally:
        C.reset_status(0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,hkv,d,bs", [(1, 1, 64, 16), (3, 4, 128, 64), (257, 3, 256, 48), (0, 2, 128, 64)])
def test_write_and_read(tokens, hkv, d, bs, dtype):
    _need_cuda()
    g = _gen(tokens + d)
    blocks = tokens // bs + 3
    kv = ops.int4_kv_cache(blocks, bs, hkv, d)
    for t in kv:
        t.copy_(torch.randint(0, 100, t.shape, generator=g, device="cuda").to(t.dtype))
    before = [t.clone() for t in kv]
    k = (3 * torch.randn(tokens, hkv, d, generator=g, device="cuda") + 1).to(dtype)
    v = (1e-3 * torch.randn(tokens, hkv, d, generator=g, device="cuda")).to(dtype)
    if tokens > 2:
        k[1] = 0.0                # constant rows: the step is 0
        v[2] = -0.375
        k[2, :, :GROUP] = 1e4     # one group far from the others
    slots = torch.randperm(blocks * bs, generator=g, device="cuda")[:tokens]
    scores = torch.rand(blocks, hkv, bs, generator=g, device="cuda")
    old = scores.clone()
    ops.gqa_cache_write_int4(kv, k, v, slots, scores)
    rk, rv = ops.gqa_cache_read_int4(kv, slots, dtype=torch.float32)
    cpu = ops.int4_kv_cache(blocks, bs, hkv, d, device="cpu")
    ops.gqa_cache_write_int4(cpu, k.cpu(), v.cpu(), slots.cpu())
    blk, off = slots // bs, slots % bs
    for t, c in zip(kv, cpu):  # every rounding is an IEEE fp32 operation: the same bits
        assert torch.equal(t[blk, :, off].cpu(), c[blk.cpu(), :, off.cpu()])
    for x, r, sc in ((k, rk, kv.k_scale), (v, rv, kv.v_scale)):
        step = sc[blk, :, off][..., 0].double().repeat_interleave(GROUP, -1)
        # half a step, and fp32 roundings of the difference, the quotient (up to 15) and the value
        tol = step / 2 * (1 + 2.0**-18) + 2.0**-22 * x.double().abs()
        assert ((r.double() - x.double()).abs() <= tol).all()
    for half in (torch.bfloat16, torch.float16):
        hk, hv = ops.gqa_cache_read_int4(kv, slots, dtype=half)
        assert torch.equal(hk, rk.to(half)) and torch.equal(hv, rv.to(half))
    mask = torch.ones(blocks, bs, dtype=torch.bool, device="cuda")
    mask[blk, off] = False
    for t, o in zip(kv, before):  # other slots stay as they were
        assert torch.equal(t.transpose(1, 2)[mask], o.transpose(1, 2)[mask])
    assert (scores[blk, :, off] == 0).all()
    assert torch.equal(scores.transpose(1, 2)[mask], old.transpose(1, 2)[mask])


def test_write_strided_and_bad_slots():
    _need_cuda()
    g = _gen(11)
    qkv = torch.randn(9, 8 * 128 + 3, generator=g, device="cuda").bfloat16()
    k = qkv[:, 3 : 3 + 256].unflatten(1, (2, 128))  # odd start: rows are not 16-byte aligned
    v = qkv[:, 512 : 512 + 256].unflatten(1, (2, 128))
    a, b = ops.int4_kv_cache(2, 16, 2, 128), ops.int4_kv_cache(2, 16, 2, 128)
    slots = torch.arange(9, device="cuda") * 3
    ops.gqa_cache_write_int4(a, k, v, slots)
    ops.gqa_cache_write_int4(b, k.contiguous(), v.contiguous(), slots)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    C = _ext.ops()
    assert C.read_status(0) == 0
    bad = slots.clone()
    bad[4], bad[5] = -1, 32
    c = ops.int4_kv_cache(2, 16, 2, 128)
    try:
        ops.gqa_cache_write_int4(c, k, v, bad)
        rk, _ = ops.gqa_cache_read_int4(c, bad)
        torch.cuda.synchronize()
        assert C.read_status(0) != 0
        assert (rk[4] == 0).all() and (rk[5] == 0).all()
        good = [0, 1, 2, 3, 6, 7, 8]
        assert torch.equal(rk[good], ops.gqa_cache_read_int4(a, slots)[0][good])
    finally:
        C.reset_status(0)


def test_refusals():
    _need_cuda()
    g = _gen(12)
    kv, table = _pool([40, 20], 2, 128, 64, g)
    lens = torch.tensor([40, 20], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 8, 128, device="cuda").bfloat16()
    ok = lambda **kw: ops.gqa_decode_int4(**{**dict(q=q, kv=kv, block_table=table, seq_lens=lens, scale=0.1), **kw})  # noqa: E731
    ok()
    for kw in (dict(q=q.float()), dict(q=q[..., :64]), dict(q=q[:, :7]), dict(q=q[:1]), dict(q=q.cpu().cuda()[..., ::2]),
               dict(seq_lens=lens.long()), dict(block_table=table.long()), dict(block_table=table[:1]),
               dict(scores=torch.zeros(3, 2, 64, device="cuda")), dict(block_table=table.cpu()),
               dict(kv=ops.Int4KV(kv.k, kv.v_scale, kv.v.int(), kv.v_scale)),
               dict(kv=ops.Int4KV(kv.k[:, :, ::2], *kv[1:])),
               dict(kv=ops.Int4KV(*(t[:, :, :8] for t in kv)))):
        with pytest.raises(RuntimeError):
            ok(**kw)
    k = torch.randn(3, 2, 128, device="cuda")
    slots = torch.arange(3, device="cuda")
    for a in ((k[:, :1], k, slots), (k, k.half(), slots), (k, k[:2], slots), (k, k, slots.int()), (k, k, slots[:2]),
              (k.double(), k.double(), slots), (k, k.cpu(), slots)):
        with pytest.raises(RuntimeError):
            ops.gqa_cache_write_int4(kv, *a)
    with pytest.raises(RuntimeError):
        ops.gqa_cache_read_int4(kv, slots, dtype=torch.float64)
    for bad in (dict(head_dim=96), dict(block_size=24)):
        with pytest.raises(ValueError):
            ops.int4_kv_cache(**{**dict(num_blocks=2, block_size=64, kv_heads=1, head_dim=64), **bad})


def test_two_streams_and_a_replayed_graph():
    """Calls on two streams at once, and captured ones replayed with other lengths, agree with plain calls."""
    _need_cuda()
    g = _gen(13)
    lens = [1500, 40, 700]
    kv, table = _pool(lens, 4, 128, 64, g)
    q = torch.randn(3, 32, 128, generator=g, device="cuda").bfloat16()
    q2 = torch.randn(3, 32, 128, generator=g, device="cuda").bfloat16()
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    short = torch.tensor([3, 0, 699], dtype=torch.int32, device="cuda")
    want = [ops.gqa_decode_int4(x, kv, table, n, 0.1) for x in (q, q2) for n in (lens_t, short)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = ops.gqa_decode_int4((q, q2)[i], kv, table, lens_t, 0.1)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[2])
    n, outs, graphs = lens_t.clone(), [], []
    scores = torch.zeros(kv.k.shape[:3], device="cuda")
    for x in (q, q2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.gqa_decode_int4(x, kv, table, n, 0.1, scores=scores))
        graphs.append(gr)
    n.copy_(short)
    for gr in graphs:
        gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[1]) and torch.equal(outs[1], want[3])
    # every head's weights sum to 1 per non-empty sequence and call: 2 calls x 2 sequences x 32 heads
    assert abs(scores.double().sum().item() - 128) < 128 * 2.0**-14
    n.copy_(lens_t)
    for s, gr in zip(streams, graphs):
        with torch.cuda.stream(s):
            gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[2])


def test_pools_past_32_bit_offsets():
    """Blocks whose codes lie more than 2^32 bytes into the cache: written, read, attended to and scored."""
    _need_cuda()
    g = _gen(21)
    blocks, bs, hkv, d = 300_000, 64, 4, 128  # 4.9 GB of codes for K and for V
    kv = ops.int4_kv_cache(blocks, bs, hkv, d)
    table = torch.tensor([[blocks - 1, 3, 270_001], [280_123, blocks - 2, 0]], dtype=torch.int32, device="cuda")
    lens = [150, 70]
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    slots = torch.cat([table[b].long()[torch.arange(n, device="cuda") // bs] * bs + torch.arange(n, device="cuda") % bs
                       for b, n in enumerate(lens)])
    k, v = (torch.randn(sum(lens), hkv, d, generator=g, device="cuda").bfloat16() for _ in range(2))
    scores = torch.zeros(blocks, hkv, bs, device="cuda")
    ops.gqa_cache_write_int4(kv, k, v, slots, scores)
    rk, rv = ops.gqa_cache_read_int4(kv, slots, dtype=torch.float32)
    assert (rk - k.float()).abs().max() < 0.4 and (rv - v.float()).abs().max() < 0.4  # half a step of about 0.3
    assert torch.equal(kv.k.view(torch.int32).ne(0).any(-1).any(-1).any(-1).nonzero()[:, 0].cpu(),
                       torch.tensor([3, 270_001, 280_123, blocks - 2, blocks - 1]))
    q = torch.randn(2, 32, d, generator=g, device="cuda").bfloat16()
    out, lse = ops.gqa_decode_int4(q, kv, table, lens_t, 0.1, scores=scores, return_lse=True)
    _check_decode(q, kv, table, lens, 0.1, out, lse, scores.double())
    new, kept = ops.kv_evict_int4(kv, scores, table, lens_t, 64, 16)
    assert new.tolist() == [64, 64] and kept[:, :, -1].tolist() == [[149] * 4, [69] * 4]
    pos = torch.arange(64, device="cuda")
    back, _ = ops.gqa_cache_read_int4(kv, table[0].long()[pos // bs] * bs + pos % bs, dtype=torch.float32)
    for h in range(hkv):
        assert torch.equal(back[:, h], rk[kept[0, h].long(), h])


def test_one_sequence_in_several_rows():
    """Rows of a batch that share blocks: equal results, and every row's weights in the scores."""
    _need_cuda()
    g = _gen(22)
    kv, table = _pool([600], 2, 128, 64, g)
    q = torch.randn(1, 8, 128, generator=g, device="cuda").bfloat16().expand(3, -1, -1)
    lens = torch.full((3,), 600, dtype=torch.int32, device="cuda")
    one, three = (torch.zeros(kv.k.shape[:3], device="cuda") for _ in range(2))
    a = ops.gqa_decode_int4(q[:1], kv, table, lens[:1], 0.1, scores=one)
    b = ops.gqa_decode_int4(q, kv, table.expand(3, -1), lens, 0.1, scores=three)
    tol = 2.0**-8 * 8 * 1.06 + 1e-3  # another split of the positions: p * step rounded to bf16 at most, steps under 1.06
    assert all((b[i].float() - a[0].float()).abs().max() <= tol for i in range(3))
    assert ((three - 3 * one).abs() <= 1e-5 * (1 + three)).all()


def test_steps_of_very_different_sizes():
    """Value steps 2^24 apart inside one head, large keys and queries near the ends of the range."""
    _need_cuda()
    g = _gen(23)
    lens = [900, 40]
    kv, table = _pool(lens, 1, 128, 64, g)
    for b, n in enumerate(lens):
        pos = torch.arange(n, device="cuda")
        blk, off = table[b].long()[pos // 64], pos % 64
        for t, spread in ((kv.v_scale, 24), (kv.k_scale, 6)):
            e = torch.randint(-spread // 2, spread // 2, (n, 1, 2, 1), generator=g, device="cuda")
            t[blk, :, off] = (t[blk, :, off].float() * torch.exp2(e.float())).bfloat16()
    for size in (1e-6, 1.0, 1e4):
        q = (size * torch.randn(2, 8, 128, generator=g, device="cuda")).bfloat16()
        lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
        out, lse = ops.gqa_decode_int4(q, kv, table, lens_t, 0.01 / size, return_lse=True)
        _check_decode(q, kv, table, lens, 0.01 / size, out, lse)
