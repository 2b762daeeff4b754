"""Cache eviction on the sm_100a kernel against a plain restatement, bit for bit."""

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


def _scores(kind, shape, g):
    s = torch.rand(shape, generator=g, device="cuda")
    if kind == "ties":  # few distinct values, both zeros
        s = (s * 5).floor() - 2
        return torch.where(s == 0, torch.copysign(torch.zeros_like(s), torch.rand(shape, generator=g, device="cuda") - 0.5), s)
    if kind == "zeros":
        return torch.zeros_like(s)
    if kind == "odd":
        s = s - 0.5
        r = torch.rand(shape, generator=g, device="cuda")
        for lo, v in ((0.9, math.nan), (0.8, math.inf), (0.7, -math.inf), (0.6, -0.0), (0.5, 1e-42)):
            s = torch.where((r > lo) & (r < lo + 0.1), v, s)
        return s
    return s**8


def _setup(lens, hkv, d, bs, width, kind, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    need = [-(-n // bs) for n in lens]
    total = sum(need) + 3
    ids = (torch.randperm(total - 1, generator=g, device="cuda") + 1).int().cpu()
    table = torch.zeros(len(lens), width or max(1, max(need)), dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = ids[at : at + k]
        at += k
    kv = ops.int4_kv_cache(total, bs, hkv, d)
    for t in (kv.k, kv.v):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, device="cuda", dtype=torch.uint8))
    for t in (kv.k_scale, kv.v_scale):
        t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
    return kv, table.cuda(), _scores(kind, kv.k.shape[:3], g)


def _plain(kv, scores, table, lens, budget, recent):
    kv, scores = [t.clone() for t in kv], scores.clone()
    hkv, bs = scores.shape[1], scores.shape[2]
    kept = torch.full((len(lens), hkv, budget), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        pos = torch.arange(n, device="cuda")
        blk, off = table[b].long()[pos // bs], pos % bs
        for h in range(hkv):
            keep = list(range(n))
            if n > budget:
                w = scores[blk, h, off].tolist()
                old = sorted(range(n - recent), key=lambda i: (-(w[i] if w[i] == w[i] else -math.inf), i))
                keep = sorted(old[: budget - recent]) + keep[n - recent :]
                src = torch.tensor(keep, device="cuda")
                for t in (*kv, scores):
                    t[blk[:budget], h, off[:budget]] = t[blk[src], h, off[src]]
            kept[b, h, : len(keep)] = torch.tensor(keep, dtype=torch.int32)
    return kv, scores, [min(n, budget) for n in lens], kept


CASES = [
    # lens, kv_heads, dim, block, budget, recent, table width
    ([100, 64, 65, 0, 1, 300], 2, 128, 64, 64, 16, None),
    ([100, 64, 65, 0, 1, 300], 2, 128, 64, 64, 0, None),
    ([100, 33], 1, 64, 16, 32, 32, None),           # the recent window alone
    ([50, 2, 1], 3, 256, 48, 1, 0, None),
    ([50, 2, 1], 3, 256, 48, 1, 1, None),
    ([700, 513, 129], 4, 128, 64, 512, 100, 40),    # a table wider than any sequence
    ([20001], 1, 128, 64, 19999, 7, None),          # eight CTAs on one sequence
    ([9000, 40], 2, 64, 64, 1031, 31, None),
    ([40] * 160 + [5000, 33], 2, 64, 16, 37, 5, None),  # one CTA each
]


@pytest.mark.parametrize("kind", ["plain", "ties", "zeros", "odd"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"n{len(c[0])}x{max(c[0])}-h{c[1]}-d{c[2]}-b{c[4]}-r{c[5]}")
def test_evict(case, kind):
    _need_cuda()
    lens, hkv, d, bs, budget, recent, width = case
    kv, table, scores = _setup(lens, hkv, d, bs, width, kind, len(lens) + budget)
    want_kv, want_scores, want_lens, want_kept = _plain(kv, scores, table, lens, budget, recent)
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    new, kept = ops.kv_evict_int4(kv, scores, table, lens_t, budget, recent)
    assert new.tolist() == want_lens
    assert torch.equal(kept.cpu(), want_kept)
    for a, b in zip(kv, want_kv):
        assert torch.equal(a, b)
    assert torch.equal(scores.view(torch.int32), want_scores.view(torch.int32))
    assert _ext.ops().read_status(0) == 0


def test_more_keys_than_shared_memory_holds():
    _need_cuda()
    lens = [10] * 297 + [60000, 55001]
    kv, table, scores = _setup(lens, 1, 64, 64, None, "ties", 3)
    want_kv, want_scores, _, want_kept = _plain(kv, scores, table, lens, 2000, 100)
    new, kept = ops.kv_evict_int4(kv, scores, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), 2000, 100)
    assert torch.equal(kept.cpu(), want_kept)
    assert all(torch.equal(a, b) for a, b in zip(kv, want_kv))
    assert torch.equal(scores.view(torch.int32), want_scores.view(torch.int32))


def test_lengths_blocks_and_refusals():
    _need_cuda()
    kv, table, scores = _setup([64, 64], 1, 64, 16, None, "plain", 5)
    lens = torch.tensor([-3, 10000], dtype=torch.int32, device="cuda")
    new, kept = ops.kv_evict_int4(kv, scores, table, lens, 20, 4)  # lengths are clamped to the table
    assert new.tolist() == [0, 20] and (kept[0] == -1).all() and kept[1, 0, -4:].tolist() == [60, 61, 62, 63]
    C = _ext.ops()
    assert C.read_status(0) == 0
    table[1, 2] = -7
    try:  # reported, and the padding block stands in
        ops.kv_evict_int4(kv, scores, table, lens, 20, 4)
        torch.cuda.synchronize()
        assert C.read_status(0) != 0
    finally:
        C.reset_status(0)
    for budget, recent in ((0, 0), (4, 5), (4, -1), (-1, -1)):
        with pytest.raises(RuntimeError):
            ops.kv_evict_int4(kv, scores, table, lens, budget, recent)
    for a in ((scores.half(), table, lens), (scores[:1], table, lens), (scores, table.long(), lens),
              (scores, table, lens.long()), (scores, table[:1], lens), (scores, table.cpu(), lens)):
        with pytest.raises(RuntimeError):
            ops.kv_evict_int4(kv, *a, 4, 1)


def test_decode_evict_decode():
    """Steps as a bounded cache takes them: write a row, attend and score, evict; a captured step replays alike."""
    _need_cuda()
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    B, heads, hkv, d, bs, budget, recent = 3, 8, 2, 64, 16, 40, 8
    kv = ops.int4_kv_cache(B * 4 + 1, bs, hkv, d)
    scores = torch.zeros(kv.k.shape[:3], device="cuda")
    table = (torch.arange(B * 4, device="cuda").view(B, 4) + 1).int()
    values = [[[] for _ in range(hkv)] for _ in range(B)]  # (k, v, score) of each cached position, on the host
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    for step in range(90):
        q = torch.randn(B, heads, d, generator=g, device="cuda").bfloat16()
        k, v = (torch.randn(B, hkv, d, generator=g, device="cuda").bfloat16() for _ in range(2))
        slots = table.long().gather(1, (lens.long() // bs)[:, None])[:, 0] * bs + lens.long() % bs
        ops.gqa_cache_write_int4(kv, k, v, slots, scores)
        rk, rv = ops.gqa_cache_read_int4(kv, slots, dtype=torch.float32)
        lens = lens + 1
        out = ops.gqa_decode_int4(q, kv, table, lens, 0.5, scores=scores)
        for b in range(B):
            for h in range(hkv):
                c = values[b][h]
                c.append([rk[b, h].double(), rv[b, h].double(), 0.0])
                s = q[b, h * 4 : h * 4 + 4].double() @ torch.stack([x[0] for x in c]).t() * 0.5
                p = torch.softmax(s, -1)
                vals = torch.stack([x[1] for x in c])
                want = p @ vals
                # p * step to bf16 (codes reach 8 steps; a step is under 0.6 here), the output to bf16
                assert ((out[b, h * 4 : h * 4 + 4].double() - want).abs() <= 2.0**-8 * (8 * 0.6 + want.abs()) + 1e-4).all()
                for x, w in zip(c, p.sum(0).tolist()):
                    x[2] += w
        if int(lens[0]) == budget + 8:
            before = scores.clone()
            lens, kept = ops.kv_evict_int4(kv, scores, table, lens, budget, recent)
            for b in range(B):
                for h in range(hkv):
                    keep = kept[b, h].tolist()
                    c = values[b][h]
                    assert keep[-recent:] == list(range(budget + 8 - recent, budget + 8))
                    # by the device's own scores (two within rounding of each other may rank either way)
                    w = before[table[b].long()].transpose(0, 1)[h].flatten()[: budget + 8 - recent].tolist()
                    assert keep[:-recent] == sorted(sorted(range(len(w)), key=lambda i: (-w[i], i))[: budget - recent])
                    assert all(abs(w[i] - c[i][2]) < 1e-3 for i in range(len(w)))
                    values[b][h] = [c[i] for i in keep]
    assert lens.tolist() == [len(values[b][0]) for b in range(B)]


def test_captured_and_replayed():
    _need_cuda()
    kv, table, scores = _setup([300, 90, 200], 2, 128, 64, None, "plain", 12)
    lens = torch.tensor([300, 90, 200], dtype=torch.int32, device="cuda")
    first = [t.clone() for t in (*kv, scores)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new, kept = ops.kv_evict_int4(kv, scores, table, lens, 96, 10)
    for n in ([300, 90, 200], [97, 96, 10]):
        for t, f in zip((*kv, scores), first):
            t.copy_(f)
        lens.copy_(torch.tensor(n))
        graph.replay()
        want_kv, want_scores, want_lens, want_kept = _plain(ops.Int4KV(*first[:4]), first[4], table, n, 96, 10)
        assert new.tolist() == want_lens and torch.equal(kept.cpu(), want_kept)
        assert all(torch.equal(a, b) for a, b in zip((*kv, scores), (*want_kv, want_scores)))


def test_scores_off_a_16_byte_boundary_are_refused():
    _need_cuda()
    kv, table, scores = _setup([64], 1, 64, 16, None, "plain", 6)
    lens = torch.tensor([64], dtype=torch.int32, device="cuda")
    shifted = torch.zeros(scores.numel() + 1, device="cuda")[1:].view(scores.shape)  # contiguous, 4 bytes off
    with pytest.raises(RuntimeError, match="16-byte"):
        ops.kv_evict_int4(kv, shifted, table, lens, 20, 4)
    with pytest.raises(RuntimeError, match="16-byte"):
        ops.gqa_decode_int4(torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda"), kv, table, lens, 1.0,
                            scores=shifted)


def test_positions_past_2_30_are_refused():
    _need_cuda()
    kv, table, scores = _setup([64], 1, 64, 16, None, "plain", 7)
    lens = torch.tensor([64], dtype=torch.int32, device="cuda")
    wide = torch.zeros(1, 2**26 + 1, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="2\\^30"):
        ops.kv_evict_int4(kv, scores, wide, lens, 4, 1)
    for budget, recent in ((2**30 + 1, 0), (2**31 - 1, 1)):
        with pytest.raises(RuntimeError, match="2\\^30"):
            ops.kv_evict_int4(kv, scores, table, lens, budget, recent)
