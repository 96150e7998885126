"""A rotation's scale that FP32 cannot hold is refused, in Python and at the C ABI, without a GPU."""

from __future__ import annotations

import pytest
import torch

from fast_mimi_amd import _native as nat
from fast_mimi_amd import training as tr

Q, F = torch.randn(1, 3, 2, 64), tr.rotary_frequencies(64)
MAX = torch.finfo(torch.float32).max


@pytest.mark.parametrize("scale", [1e39, -1e39, 1e300, float("inf"), -float("inf"), float("nan")])
def test_python(scale):
    for call in (tr.rotary, tr.rotary_forward, tr.rotary_backward):
        with pytest.raises(ValueError, match="scale must be finite"):
            call(Q, None, F, scale=scale)
    for fits in (MAX, -MAX, 0.0):
        with pytest.raises(ValueError, match="ROCm GPU"):  # as far as a CPU goes
            tr.rotary(Q, None, F, scale=fits)


@pytest.mark.skipif(not nat.LIBRARY_PATH.is_file(), reason="library not built")
def test_abi():
    P = 0x10000  # never dereferenced

    def call(scale):
        return nat.library().fm_rotary(P, 64, 64, 64, 4, P, 64, 64, 64, 2, P, P, 3, 8, 0, 0, 3, 64, 64, 0, scale, 0, 1, P, P, None)

    assert call(1e39) == call(-float("inf")) == call(float("nan")) == 1000 and call(MAX) == call(0.0) == 0
