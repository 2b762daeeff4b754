"""Measured cases of the quantised Attention-role operators.

Operators (``afd_plugin_b200.ops``):

* ``gqa_cache_write_int4`` / ``gqa_cache_read_int4``: K / V rows into the paged 4-bit cache and back
* ``gqa_decode_int4``: single-token attention over that cache, optionally adding each cached
  position's attention weight to its score
* ``kv_evict_int4``: keep the recent and the most attended positions, compact the cache in place
* ``int8_linear``: 8-bit integer product with a scale per token and per output channel

The 4-bit cache holds, per block, KV head and position, ``d / 2`` bytes of codes (dim ``2 i`` in the
low nibble of byte ``i``) and per 64 dims a bf16 ``(step, zero)``; a code ``c`` stands for
``zero + c * step``.  Block 0 is the padding block.
"""

import math

import torch

own = False

BLOCK = 64
GROUP = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # two chat requests early in their answers, Qwen3-30B heads: launch latency is all there is
        {"name": "decode short", "op": "decode", "batch": 2, "heads": 32, "kv_heads": 4, "dim": 128,
         "shortest": 1, "longest": 61, "dtype": "bf16"},
        # a full serving batch with ragged lengths, Qwen3-Next heads (two KV heads of 256)
        {"name": "decode ragged batch", "op": "decode", "batch": 256, "heads": 16, "kv_heads": 2, "dim": 256,
         "shortest": 1, "longest": 4001, "dtype": "bf16"},
        # long documents: the cache does not fit L2 many times over
        {"name": "decode long", "op": "decode", "batch": 16, "heads": 32, "kv_heads": 4, "dim": 128,
         "shortest": 50001, "longest": 131072, "dtype": "bf16"},
        # decode under a cache budget, multi-head attention (DeepSeek V1), fp16 activations
        {"name": "scored multi-head", "op": "scored", "batch": 16, "heads": 16, "kv_heads": 16, "dim": 128,
         "shortest": 777, "longest": 2050, "dtype": "fp16"},
        # decode under a cache budget, 16 query heads on each KV head, long contexts
        {"name": "scored wide group", "op": "scored", "batch": 4, "heads": 64, "kv_heads": 4, "dim": 128,
         "shortest": 20000, "longest": 32768, "dtype": "bf16"},
        # the K / V rows of one decode step
        {"name": "write step", "op": "write", "tokens": 64, "kv_heads": 4, "dim": 128, "dtype": "bf16"},
        # the K / V rows of a prefill chunk, read back for its attention
        {"name": "write prefill", "op": "write", "tokens": 16001, "kv_heads": 8, "dim": 128, "dtype": "bf16"},
        # a few requests just over their budget
        {"name": "evict few", "op": "evict", "batch": 3, "kv_heads": 4, "dim": 128, "shortest": 1000,
         "longest": 1153, "budget": 1024, "recent": 128},
        # a batch of long prompts cut to a quarter
        {"name": "evict long", "op": "evict", "batch": 32, "kv_heads": 4, "dim": 128, "shortest": 20001,
         "longest": 32768, "budget": 8192, "recent": 1024},
        # fused q / k / v projection of one small decode batch
        {"name": "int8 few tokens", "op": "int8", "tokens": 5, "n": 5120, "k": 2048, "dtype": "bf16"},
        # down projection of a dense layer at a full decode batch (long contraction, ragged tile edges)
        {"name": "int8 decode batch", "op": "int8", "tokens": 256, "n": 2048, "k": 10944, "dtype": "bf16"},
        # gate and up projection of a DeepSeek-V3 dense layer over a prefill step
        {"name": "int8 prefill", "op": "int8", "tokens": 4099, "n": 36864, "k": 7168, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("decode", "scored", "write", "evict", "int8"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    kv_heads = rng.choice((1, 2, 4, 8, 16))
    if op in ("decode", "scored"):
        dim = rng.choice((64, 128, 128, 256))
        heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 5, 7, 8, 12, 16) if g * kv_heads <= 64])
        batch = _log(rng, 1, 256)
        # codes of the pool stay below those of the largest listed case
        longest = _log(rng, 1, min(131072, 500_000_000 // (batch * kv_heads * dim)))
        return {"op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "shortest": rng.randint(0, longest), "longest": longest, "dtype": dtype}
    if op == "write":
        return {"op": op, "tokens": _log(rng, 1, 16001), "kv_heads": min(kv_heads, 8),
                "dim": rng.choice((64, 128)), "dtype": dtype}
    if op == "evict":
        batch = _log(rng, 1, 32)
        longest = _log(rng, 65, 32768)
        budget = rng.randint(1, longest)
        return {"op": op, "batch": batch, "kv_heads": min(kv_heads, 4), "dim": rng.choice((64, 128)),
                "shortest": rng.randint(1, longest), "longest": longest, "budget": budget,
                "recent": rng.randint(0, budget)}
    return {"op": op, "tokens": _log(rng, 1, 4099), "n": _log(rng, 16, 36864), "k": 16 * _log(rng, 4, 448),
            "dtype": dtype}


def _lengths(case):
    b, lo, hi = case["batch"], case["shortest"], case["longest"]
    return [hi - (hi - lo) * i // max(1, b - 1) for i in range(b)]


# ----------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _filled_pool(blocks, kv_heads, dim, g, spread):
    """A pool of quantised rows, made like the cache write makes them, in slices that stay small."""
    codes = torch.empty(blocks, kv_heads, BLOCK, dim // 2, dtype=torch.uint8, device="cuda")
    scale = torch.empty(blocks, kv_heads, BLOCK, dim // GROUP, 2, dtype=torch.bfloat16, device="cuda")
    per = max(1, (1 << 26) // (kv_heads * BLOCK * dim))
    # a few dims of a head are much larger than the rest, as in real keys
    amp = 1 + spread * (torch.rand(kv_heads, 1, dim, generator=g, device="cuda") > 0.95).float()
    for lo in range(0, blocks, per):
        n = min(per, blocks - lo)
        x = torch.randn(n, kv_heads, BLOCK, dim, generator=g, device="cuda") * amp
        codes[lo : lo + n], scale[lo : lo + n] = _quantise(x.bfloat16())
    return codes, scale


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    dt = DTYPES[case.get("dtype", "bf16")]
    if op == "int8":
        t, n, k = case["tokens"], case["n"], case["k"]
        x = torch.randn(t, k, generator=g, device="cuda")
        x = x * (1 + 4 * (torch.rand(k, generator=g, device="cuda") > 0.99).float())  # outlier channels
        w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
        ws = (0.5 + torch.rand(n, generator=g, device="cuda")) / (73.0 * math.sqrt(k))
        return {"op": op, "x": x.to(dt), "w": w, "w_scale": ws}
    hkv, d = case["kv_heads"], case["dim"]
    if op == "write":
        t = case["tokens"]
        blocks = 2 * -(-t // BLOCK) + 1
        k = torch.randn(t, hkv, d, generator=g, device="cuda").to(dt)
        v = torch.randn(t, hkv, d, generator=g, device="cuda").to(dt)
        slots = torch.randperm((blocks - 1) * BLOCK, generator=g, device="cuda")[:t] + BLOCK
        return {"op": op, "k": k, "v": v, "slots": slots, "kv": _empty_pool(blocks, hkv, d)}
    lens = _lengths(case)
    order = torch.randperm(len(lens), generator=g, device="cuda")
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")[order]
    width = max(1, -(-max(lens) // BLOCK))
    need = (lens_t.long() + BLOCK - 1) // BLOCK
    total = sum(-(-n // BLOCK) for n in lens)
    ids = (torch.randperm(total, generator=g, device="cuda") + 1).to(torch.int32)
    table = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    table[torch.arange(width, device="cuda")[None, :] < need[:, None]] = ids
    kv = _filled_pool(total + 1, hkv, d, g, 3.0) + _filled_pool(total + 1, hkv, d, g, 0.0)
    state = {"op": op, "kv": kv, "table": table, "lens": lens_t}
    if op == "evict":
        # accumulated weights: heavy-tailed, many exact zeros (positions that no query attended to)
        s = torch.rand(total + 1, hkv, BLOCK, generator=g, device="cuda")
        state |= {"scores": torch.where(s < 0.1, 0.0, s**8), "budget": case["budget"], "recent": case["recent"]}
        return state
    q = 1.5 * torch.randn(len(lens), case["heads"], d, generator=g, device="cuda")
    state |= {"q": q.to(dt), "scale": 1 / math.sqrt(d)}
    if op == "scored":
        state["scores"] = torch.rand(total + 1, hkv, BLOCK, generator=g, device="cuda") / 16
    return state


def _empty_pool(blocks, hkv, d):
    def one():
        return (torch.zeros(blocks, hkv, BLOCK, d // 2, dtype=torch.uint8, device="cuda"),
                torch.zeros(blocks, hkv, BLOCK, d // GROUP, 2, dtype=torch.bfloat16, device="cuda"))

    return one() + one()


# ------------------------------------------------------------- plain forms
def _bf16_up(x):
    """The smallest bf16 value >= x, as fp32 (x >= 0)."""
    return ((x.view(torch.int32) + 0xFFFF) & -0x10000).view(torch.float32)


def _bf16_down(x):
    """The largest bf16 value <= x, as fp32."""
    b = x.view(torch.int32)
    return torch.where(b < 0, (b + 0xFFFF) & -0x10000, b & -0x10000).view(torch.float32)


def _quantise(x):
    """codes ``[..., d / 2]`` uint8 and ``(step, zero) [..., d / 64, 2]`` bf16 of rows ``x [..., d]``."""
    g = x.float().unflatten(-1, (-1, GROUP))
    zero = _bf16_down(g.amin(-1, keepdim=True))
    # divided by a tensor: by a number it would be a product with the rounded reciprocal
    step = _bf16_up((g.amax(-1, keepdim=True) - zero) / g.new_full((1,), 15.0))
    c = torch.where(step > 0, (g - zero) / step, torch.zeros_like(g)).round().clamp(0, 15)
    c = c.to(torch.uint8).flatten(-2)
    return c[..., 0::2] | (c[..., 1::2] << 4), torch.cat([step, zero], -1).bfloat16()


def _values(codes, scale):
    """fp32 values of packed rows."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    s = scale.float()
    return (s[..., 1:] + c.unflatten(-1, (-1, GROUP)) * s[..., :1]).flatten(-2)


def _rows(codes, scale, table):
    """fp32 rows ``[batch, kv_heads, positions, dim]`` of every sequence."""
    t = table.long()
    return _values(codes[t].transpose(1, 2).flatten(2, 3), scale[t].transpose(1, 2).flatten(2, 3))


def _attend(s):
    k = _rows(s["kv"][0], s["kv"][1], s["table"])
    q = s["q"].float().unflatten(1, (k.shape[1], -1))
    z = (q @ k.transpose(2, 3)) * s["scale"]
    del k
    valid = (torch.arange(z.shape[-1], device=z.device) < s["lens"][:, None])[:, None, None, :]
    z = torch.where(valid, z, -math.inf)
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(torch.isinf(top), 0.0, top))
    total = e.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).flatten(1)
    p = e / torch.where(total > 0, total, 1.0)
    o = p @ _rows(s["kv"][2], s["kv"][3], s["table"])
    return o.flatten(1, 2).to(s["q"].dtype), lse, p


def _slots(s, positions, hkv):
    """Flat ``(block, head, offset)`` index of ``positions [batch, heads, n]``."""
    blk = s["table"].long().gather(1, (positions // BLOCK).flatten(1)).view_as(positions)
    head = torch.arange(hkv, device=blk.device)[None, :, None]
    return (blk * hkv + head) * BLOCK + positions % BLOCK


def _add_scores(s, p):
    b, hkv, _, n = p.shape
    at = _slots(s, torch.arange(n, device=p.device).expand(b, hkv, n), hkv)
    s["scores"].view(-1).index_add_(0, at.flatten(), p.sum(2).flatten())


def _evict(s):
    hkv, width = s["scores"].shape[1], s["table"].shape[1] * BLOCK
    b, budget, lens = len(s["lens"]), s["budget"], s["lens"].long()[:, None, None]
    pos = torch.arange(width, device=lens.device).expand(b, hkv, width)
    key = s["scores"].view(-1)[_slots(s, pos, hkv)]
    key = torch.where(pos >= lens - s["recent"], math.inf, key)
    key = torch.where(pos >= lens, -math.inf, key)
    new = s["lens"].clamp(max=budget)
    take = min(budget, width)
    kept = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :take]
    kept = torch.where(torch.arange(take, device=lens.device) < new[:, None, None], kept, width).sort(-1).values
    real = kept < width
    src = _slots(s, kept.clamp(max=width - 1), hkv)[real]
    dst = _slots(s, pos[..., :take], hkv)[real]
    for t in s["kv"] + (s["scores"],):
        flat = t.view(t.shape[0] * hkv * BLOCK, -1)
        flat[dst] = flat[src]
    out = torch.full((b, hkv, budget), -1, dtype=torch.int32, device=lens.device)
    out[..., :take] = torch.where(real, kept, -1).int()
    return new, out


def _int8(x):
    amax = x.float().abs().amax(-1, keepdim=True).clamp(min=2.0**-100)
    top = amax.new_full((1,), 127.0)
    return (x.float() * (top / amax)).round().clamp(-127, 127), amax / top


def run(state):
    s = state
    op = s["op"]
    if own:
        from afd_plugin_b200 import ops

        if op == "int8":
            return ops.int8_linear(s["x"], s["w"], s["w_scale"])
        kv = ops.Int4KV(*s["kv"])
        if op == "write":
            ops.gqa_cache_write_int4(kv, s["k"], s["v"], s["slots"])
            return ops.gqa_cache_read_int4(kv, s["slots"], dtype=torch.float32)
        if op == "decode":
            return ops.gqa_decode_int4(s["q"], kv, s["table"], s["lens"], s["scale"], return_lse=True)
        if op == "scored":
            o = ops.gqa_decode_int4(s["q"], kv, s["table"], s["lens"], s["scale"], scores=s["scores"])
            return o, s["scores"]
        new, kept = ops.kv_evict_int4(kv, s["scores"], s["table"], s["lens"], s["budget"], s["recent"])
        return new, kept, s["kv"], s["scores"]
    if op == "int8":
        q, xs = _int8(s["x"])
        return ((q @ s["w"].float().t()) * (xs * s["w_scale"])).to(s["x"].dtype)
    if op == "write":
        blk, off = s["slots"] // BLOCK, s["slots"] % BLOCK
        for i, x in ((0, s["k"]), (2, s["v"])):
            s["kv"][i][blk, :, off], s["kv"][i + 1][blk, :, off] = _quantise(x)
        return tuple(_values(s["kv"][i][blk, :, off], s["kv"][i + 1][blk, :, off]) for i in (0, 2))
    if op == "decode":
        return _attend(s)[:2]
    if op == "scored":
        o, _, p = _attend(s)
        _add_scores(s, p)
        return o, s["scores"]
    return (*_evict(s), s["kv"], s["scores"])


# ------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "int8":
        t, n, k = case["tokens"], case["n"], case["k"]
        return {"bytes": 2 * t * k + n * k + 4 * n + 2 * t * n, "flops": 2 * t * n * k}
    hkv, d = case["kv_heads"], case["dim"]
    row = d // 2 + 4 * d // GROUP  # one packed K or V row
    if op == "write":
        # K and V in, packed rows out, and the packed rows' values out
        t = case["tokens"]
        return {"bytes": t * (2 * hkv * (2 * d + row + 4 * d) + 8), "flops": 0}
    lens = _lengths(case)
    if op == "evict":
        # every score once; the kept rows (K, V, score) read and written
        over = [n for n in lens if n > case["budget"]]
        return {"bytes": hkv * (4 * sum(over) + len(over) * case["budget"] * (2 * (2 * row + 4) + 4)) + 8 * len(lens),
                "flops": 0}
    total, b, hq = sum(lens), case["batch"], case["heads"]
    bytes_ = total * hkv * 2 * row + 4 * b * hq * d + 4 * b * -(-case["longest"] // BLOCK) + 4 * b
    if op == "scored":
        bytes_ += total * hkv * 8
    return {"bytes": bytes_, "flops": 4 * total * hq * d}


# ------------------------------------------------------------------ exact
def _ceil8(x):
    """Rounded up to 8 significant bits (x >= 0)."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.ceil(m * 256), e - 8)


def _exact_values(x):
    """What the stored form of rows ``x`` stands for; the definition rounds its steps to 32 bits."""
    g = x.double().reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
    zero = torch.where(lo < 0, -_ceil8(lo.abs()), 0.0)
    m, e = torch.frexp(lo.clamp(min=0))
    zero = torch.where(lo > 0, torch.ldexp(torch.floor(m * 256), e - 8), zero)
    r32 = lambda v: v.float().double()  # noqa: E731
    step = _ceil8(r32(r32(hi - zero) / 15))
    c = torch.round(r32(r32(g - zero) / torch.where(step > 0, step, 1.0))).clamp(0, 15) * (step > 0)
    return (zero + c * step).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "int8":
        x = s["x"].double()
        amax = x.abs().max(1, keepdim=True).values.clamp(min=2.0**-100)
        r = (127 / amax).float().double()  # the definition multiplies by the 32-bit reciprocal
        q = torch.round((x * r).float().double()).clamp(-127, 127)
        return (q @ s["w"].double().t()) * ((amax / 127) * s["w_scale"].double())
    if op == "write":
        return _exact_values(s["k"]), _exact_values(s["v"])
    if op == "evict":
        return _exact_evict(s)
    hkv = case["kv_heads"]
    group = case["heads"] // hkv
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    scores = s["scores"].double() if op == "scored" else None
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        blocks = s["table"][b, : -(-n // BLOCK)].long()
        for h in range(hkv):
            k, v = (_unpack64(s["kv"][i], s["kv"][i + 1], blocks, h)[:n] for i in (0, 2))
            hs = slice(h * group, (h + 1) * group)
            z = s["q"][b, hs].double() @ k.t() * s["scale"]
            lse[b, hs] = torch.logsumexp(z, -1)
            p = torch.exp(z - lse[b, hs, None])
            o[b, hs] = p @ v
            if scores is not None:
                w = torch.zeros(len(blocks) * BLOCK, dtype=torch.float64, device="cuda")
                w[:n] = p.sum(0)
                scores[blocks, h] += w.view(-1, BLOCK)
    return (o, lse) if op == "decode" else (o, scores)


def _unpack64(codes, scale, blocks, h):
    c = codes[blocks, h].reshape(-1, codes.shape[-1]).to(torch.int16)
    c = torch.stack((c % 16, c // 16), 2).reshape(c.shape[0], -1, GROUP).double()
    s = scale[blocks, h].reshape(c.shape[0], -1, 2).double()
    return (s[:, :, 1:] + s[:, :, :1] * c).reshape(c.shape[0], -1)


def _exact_evict(s):
    """Scores after the move, in 64 bits; what is only moved or counted has no value of its own here."""
    scores = s["scores"].double()
    before = scores.clone()
    for b, n in enumerate(s["lens"].tolist()):
        if n <= s["budget"]:
            continue
        pos = torch.arange(n, device="cuda")
        for h in range(scores.shape[1]):
            blk = s["table"][b].long()[pos // BLOCK]
            w = before[blk, h, pos % BLOCK]
            old = n - s["recent"]
            # rank by (score, earlier position first): a stable sort of the negated scores
            best = torch.sort(-w[:old], stable=True).indices[: s["budget"] - s["recent"]]
            keep = torch.cat([best, pos[old:]]).sort().values
            at = pos[: len(keep)]
            scores[blk[at], h, at % BLOCK] = w[keep]
    return None, None, None, scores
