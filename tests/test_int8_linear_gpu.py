"""The int8 linear layer on the sm_100a kernels: exact integer sums, scales in fp32."""

import pytest
import torch

from afd_plugin_b200 import ops
from afd_plugin_b200.ops import _ext
from afd_plugin_b200.ops import reference as ref

pytestmark = pytest.mark.gpu


def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    assert _ext.load(), "extension not built"


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _check(x, w, ws, y):
    q, s = ref.int8_quantize(x.cpu())  # IEEE fp32 operations: the same on the CPU
    want = (q.cuda().double() @ w.double().t()) * s.cuda().double()[:, None] * ws.double()[None, :]
    # fp32 roundings of the sum, the scales' product and the result, then the output's own
    tol = want.abs() * (torch.finfo(y.dtype).eps / 2 + 4 * 2.0**-24) + torch.finfo(y.dtype).smallest_normal
    err = (y.double() - want).abs()
    assert (err <= tol).all(), (err / tol).max().item()


SHAPES = [  # tokens, n, k
    (1, 1, 16), (3, 7, 48), (8, 32, 128), (5, 5120, 2048), (1, 130, 10944),   # K split over a cluster
    (127, 100, 144), (128, 128, 1024), (129, 257, 528), (256, 2048, 2736),
    (300, 1000, 272), (20, 20000, 256),                                        # one pass of 128-wide tiles
    (1100, 4500, 400), (2500, 2100, 640), (4099, 1030, 128),                   # 256 x 256 on pairs of SMs
    (129, 19000, 144), (700, 7000, 2048),
    (100, 40000, 144), (1, 76000, 64),                                         # 128 x 256, several tiles a CTA
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_linear(shape, dtype):
    _need_cuda()
    t, n, k = shape
    g = _gen(t + n + k)
    x = torch.randn(t, k, generator=g, device="cuda").to(dtype)
    if t > 2:
        x[1] = 0
        x[2] *= 1e-3
    w = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    ws = torch.rand(n, generator=g, device="cuda") / 100
    y = ops.int8_linear(x, w, ws)
    assert y.dtype == dtype and _ext.ops().read_status(0) == 0
    _check(x, w, ws, y)


def test_quantize_strided_odd_values_and_weights():
    _need_cuda()
    g = _gen(1)
    base = torch.randn(9, 533, generator=g, device="cuda").bfloat16()
    x = base[:, 5:517]  # rows that are not 16-byte aligned
    x[0, 3], x[1, 4], x[2] = float("inf"), float("nan"), 0
    x[3] = 1e-38
    q, s = ops.int8_quantize(x)
    cq, cs = ops.int8_quantize(x.cpu())
    fine = torch.isfinite(x).all(1).cpu()
    assert torch.equal(q.cpu()[fine], cq[fine]) and torch.equal(s.cpu()[fine], cs[fine])
    assert not torch.isfinite(s[:2]).any()
    w, ws = ops.int8_quantize(torch.randn(70, 512, generator=g, device="cuda"))
    y = ops.int8_linear(x, w, ws, out_dtype=torch.float32)
    assert y.dtype == torch.float32 and torch.isnan(y[1]).all() and not torch.isfinite(y[0]).any()
    _check(x[2:], w, ws, y[2:])
    empty = ops.int8_linear(x[:0], w, ws)
    assert empty.shape == (0, 70)


def test_largest_sums():
    """k = 131072 with every product at its largest: the int32 sums stay in range."""
    _need_cuda()
    x = torch.ones(2, 131072, device="cuda")
    w = torch.full((40, 131072), -128, dtype=torch.int8, device="cuda")
    ws = torch.ones(40, device="cuda")
    _check(x, w, ws, ops.int8_linear(x, w, ws))


def test_refusals():
    _need_cuda()
    x = torch.randn(4, 64, device="cuda")
    w = torch.zeros(8, 64, dtype=torch.int8, device="cuda")
    ws = torch.ones(8, device="cuda")
    ops.int8_linear(x, w, ws)
    for a in ((x[:, :24], w[:, :24].contiguous(), ws), (x, w[:, :48].contiguous(), ws), (x, w.float(), ws), (x, w, ws[:7]),
              (x, w, ws.double()), (x, w.cpu(), ws), (x[0], w, ws), (x.double(), w, ws), (x, w[:, :32], ws),
              (x, w.t().contiguous().t(), ws), (x, w[:0], ws[:0]), (x.t().contiguous().t(), w, ws)):
        with pytest.raises(RuntimeError):
            ops.int8_linear(*a)
    with pytest.raises(RuntimeError):
        ops.int8_linear(x, w, ws, out_dtype=torch.float64)
    with pytest.raises(RuntimeError):
        ops.int8_quantize(torch.zeros(1, 131088, device="cuda"))


def test_streams_and_replayed_graph():
    _need_cuda()
    g = _gen(2)
    w, ws = ops.int8_quantize(torch.randn(512, 1024, generator=g, device="cuda"))
    xs = [torch.randn(t, 1024, generator=g, device="cuda").bfloat16() for t in (3, 200, 1500)]
    want = [ops.int8_linear(x, w, ws) for x in xs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [ops.int8_linear(x, w, ws) for x in xs]
    graph.replay()
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(ops.int8_linear(x, w, ws))
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, outs):
        assert torch.equal(a, b) and torch.equal(a, c)
    for x in xs:
        x.mul_(-1)
    graph.replay()
    for a, c in zip(want, outs):
        assert torch.equal(-a, c)
