"""What a module's parameters do in the 8-bit operators: scales that require a gradient are refused like values."""

from __future__ import annotations

import pytest
import torch

from fast_mimi_amd import quantized as qz

X8, W8 = torch.zeros(4, 256).to(torch.float8_e4m3fn), torch.zeros(100, 256).to(torch.float8_e4m3fn)
XS, WS = (torch.full((n, 2), 127, dtype=torch.uint8).view(torch.float8_e8m0fnu) for n in (4, 1))


@pytest.mark.parametrize("which", [1, 3])
def test_scales_that_require_a_gradient_are_refused(which):
    args = [X8, XS, W8, WS]
    args[which] = torch.nn.Parameter(args[which])
    with pytest.raises(RuntimeError, match="no gradient"):
        qz.linear(*args)
    with torch.no_grad(), pytest.raises(ValueError, match="ROCm GPU"):  # as far as a CPU goes
        qz.linear(*args)
