"""Cache groups with values that are not finite read back as NaN, and only they."""

import math

import pytest
import torch

from afd_plugin_b200 import ops
from afd_plugin_b200.ops import reference as ref

INF, NAN = math.inf, math.nan


def rows(dtype: torch.dtype) -> torch.Tensor:
    """``[rows, 1, 128]``: the second group of a row is spoilt, in another way each, the first is not."""
    x = torch.randn(10, 1, 128, generator=torch.Generator().manual_seed(5))
    x[0, 0, 64] = NAN
    x[1, 0, 127] = -NAN
    x[2, 0, 70] = INF
    x[3, 0, 71] = -INF
    x[4, 0, 80:83] = torch.tensor([INF, NAN, -INF])
    x[5, 0, 64:] = INF
    x[6, 0, 64:] = -INF
    x[7, 0, 64:] = NAN
    x[8, 0, 90], x[8, 0, 91] = INF, -INF
    x = x.to(dtype)
    big = torch.finfo(dtype).max if dtype != torch.float16 else INF
    x[9, 0, 64], x[9, 0, 65] = big, -big  # the range overflows fp32
    return x


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_groups_that_are_not_finite_read_back_as_nan(dtype):
    x = rows(dtype)
    kv = ops.int4_kv_cache(1, 16, 1, 128, device="cpu")
    ops.gqa_cache_write_int4(kv, x, x, torch.arange(10))
    for back in ops.gqa_cache_read_int4(kv, torch.arange(10), dtype=torch.float32):
        assert back[:, :, 64:].isnan().all()
        assert back[:, :, :64].isfinite().all()
        assert (back[:, :, :64] - x[:, :, :64].float()).abs().max() < 0.4  # half a step of about 0.3


def test_any_nan_payload():
    x = torch.zeros(4, 64)
    x[:, 3] = torch.tensor([0x7FFFFFFF, 0x7F800001, -1, -0x7FFFFF], dtype=torch.int32).view(torch.float32)
    codes, scale = ref.int4_quantize(x)
    assert (codes == 0).all() and scale.isnan().all()


def test_nan_pairs_have_one_encoding():
    """The stored pair is the quiet NaN 0x7FC0 in both halves, whatever the vector unit makes of a cast."""
    for n in (1, 40):  # short and long rows take different paths of a cast
        x = torch.zeros(n, 64)
        x[:, 5] = NAN
        _, scale = ref.int4_quantize(x)
        assert (scale.view(torch.int16) == 0x7FC0).all()
