"""Refusals of the extension that name a number raise; they must not end the process."""

import pytest
import torch

from afd_plugin_b200.ops import _ext


def test_the_extension_uses_the_shared_cpp_runtime():
    """A static copy of the C++ runtime beside PyTorch's crashes where it formats a number."""
    path = _ext.library_path()
    if path is None:
        pytest.skip("extension not built")
    with open(path, "rb") as f:
        assert b"libstdc++.so.6\0" in f.read()  # named in the dynamic section


@pytest.mark.gpu
def test_refusals_that_name_a_number():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    C = _ext.ops()
    with pytest.raises(RuntimeError, match="multiple of 8"):
        C.rms_norm(torch.zeros(2, 12, device="cuda", dtype=torch.bfloat16),
                   torch.ones(12, device="cuda", dtype=torch.bfloat16), 1e-6)
    with pytest.raises(RuntimeError, match="multiple of 4"):
        C.silu_and_mul(torch.zeros(2, 12, device="cuda"))
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        C.argmax_rows(torch.zeros(2, 16, device="cuda", dtype=torch.float64))
