"""The layers' attention over the 4-bit cache, prompts and single tokens: GPU against the CPU path, same inputs."""

import math

import pytest
import torch

from afd_plugin_b200 import ops
from afd_plugin_b200.models.layers import AttentionMetadata, Int4Layer, _attend_int4
from afd_plugin_b200.ops import _ext

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("heads,hkv,d,bs", [(8, 2, 128, 16), (4, 4, 64, 32), (6, 1, 256, 16)])
def test_prompts_then_single_tokens(heads, hkv, d, bs, scored, dtype):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    assert _ext.load(), "extension not built"
    g = torch.Generator().manual_seed(heads + d)
    lens, width = [41, 1, 90], 8
    table = (torch.randperm(3 * width, generator=g).view(3, width) + 1).int()
    scale = 1 / math.sqrt(d)

    def layer(dev):
        kv = ops.int4_kv_cache(3 * width + 1, bs, hkv, d, device=dev)
        return Int4Layer(kv, torch.zeros(kv.k.shape[:3], device=dev) if scored else None)

    gpu, cpu = layer("cuda"), layer("cpu")
    half = torch.finfo(dtype).eps / 2

    def step(positions, seq_of, prefill):
        """One step of tokens at ``positions`` of sequences ``seq_of`` on both devices; the outputs agree."""
        n = len(positions)
        pos, seqs = torch.tensor(positions), torch.tensor(seq_of)
        slots = table.long()[seqs, pos // bs] * bs + pos % bs
        q = torch.randn(n, heads, d, generator=g).to(dtype)
        k, v = (torch.randn(n, hkv, d, generator=g).to(dtype) for _ in range(2))
        out = {}
        for dev, cache in (("cuda", gpu), ("cpu", cpu)):
            meta = AttentionMetadata(
                positions=pos.to(dev), slot_mapping=slots.to(dev), block_table=table.to(dev),
                seq_lens=torch.tensor([p + 1 for p in positions], dtype=torch.int32, device=dev) if not prefill
                else torch.tensor(lens, dtype=torch.int32, device=dev),
                is_decode=not prefill, prefill_seqs=prefill)
            out[dev] = _attend_int4(q.to(dev), k.to(dev), v.to(dev), meta, cache, scale).double().cpu()
        for a, b in zip(gpu.kv, cpu.kv):
            assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))
        # Each side's output rounding; 2^-11 for p * step in fp16, of 8 steps at most, which are below 2 max|v| (4.5
        # for so many normal values); logits under 30 with d / 16 + 8 fp32 roundings each way.
        off = 2 * (d / 16 + 8) * 2.0**-24 * 30 + 2.0**-16
        tol = 2 * half * out["cpu"].abs() + (2.0**-11 + 2 * off) * 2 * 5.5
        assert ((out["cuda"] - out["cpu"]).abs() <= tol).all()

    prefill, flat, seqs = [], [], []
    for b, n in enumerate(lens):
        prefill.append((len(flat), len(flat) + n, b))
        flat += range(n)
        seqs += [b] * n
    step(flat, seqs, prefill)
    for t in range(6):
        step([n + t for n in lens], [0, 1, 2], None)
    if scored:
        w, want = gpu.scores.double().cpu(), cpu.scores.double()
        # a weight of at most group x queries, each off by its logit's error
        assert ((w - want).abs() <= (heads // hkv) * (max(lens) + 6) * 2.0**-14).all()
        for b, n in enumerate(lens):  # each query spreads 1 per query head over its sequence
            total = w[table[b].long()].sum((0, 2))
            assert (total - (heads // hkv) * (n + 6)).abs().max() <= (heads // hkv) * (n + 6) * 2.0**-14
    assert _ext.ops().read_status(0) == 0
