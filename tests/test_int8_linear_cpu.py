"""The int8 linear layer on CPU: its definition in exact arithmetic, and the refusals."""

from fractions import Fraction

import pytest
import torch

from afd_plugin_b200 import ops


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_definition(dtype):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 32, generator=g).to(dtype)
    x[1], x[2] = 0, x[2] * 1e-4
    q, s = ops.int8_quantize(x)
    for row, c, scale in zip(x.double().tolist(), q.tolist(), s.double().tolist()):
        amax = max(max(abs(v) for v in row), 2.0**-100)
        assert abs(scale - amax / 127) <= scale * 2.0**-24
        for v, i in zip(row, c):
            # rint of v * 127 / amax, up to two fp32 roundings at a tie
            assert abs(Fraction(v) * 127 / Fraction(amax) - i) <= Fraction(1, 2) + Fraction(1, 2**16)
    w, ws = ops.int8_quantize(torch.randn(7, 32, generator=g))
    y = ops.int8_linear(x, w, ws, out_dtype=torch.float32)
    for t in range(5):
        for n in range(7):
            acc = sum(a * b for a, b in zip(q[t].tolist(), w[n].tolist()))
            want = acc * s[t].double().item() * ws[n].double().item()
            assert abs(y[t, n].item() - want) <= abs(want) * 4 * 2.0**-24


def test_rounding_error_of_the_product():
    """Against the unquantised product: each operand is off by at most half a step of its row."""
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(6, 64, generator=g), torch.randn(9, 64, generator=g)
    q, s = ops.int8_quantize(w)
    y = ops.int8_linear(x, q, s).double()
    dx, dw = x.double().abs().amax(1) / 254 * (1 + 2.0**-16), w.double().abs().amax(1) / 254 * (1 + 2.0**-16)
    bound = (x.double().abs().sum(1)[:, None] * dw[None] + w.double().abs().sum(1)[None] * dx[:, None]
             + 64 * dx[:, None] * dw[None])
    assert ((y - x.double() @ w.double().t()).abs() <= bound).all()


def test_refusals():
    x, w, ws = torch.randn(4, 64), torch.zeros(8, 64, dtype=torch.int8), torch.ones(8)
    for a in ((x[:, :24], w[:, :24].contiguous(), ws), (x, w[:, :48].contiguous(), ws), (x, w.float(), ws),
              (x, w, ws[:7]), (x, w, ws.double()), (x[0], w, ws), (x.double(), w, ws), (x, w[:0], ws[:0])):
        with pytest.raises(ValueError):
            ops.int8_linear(*a)
    with pytest.raises(ValueError):
        ops.int8_linear(x, w, ws, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        ops.int8_quantize(torch.zeros(1, 131088))
    assert ops.int8_linear(x[:0], w, ws).shape == (0, 8)
