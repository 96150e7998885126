"""What a module's parameters do in the 8-bit operators: scales that require a gradient are refused like values, and
frozen parameters reach the kernels as plain tensors do."""

from __future__ import annotations

import pytest
import torch

from fast_mimi_amd import _native as nat
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


@pytest.mark.gpu
def test_frozen_parameters_take_the_direct_call(monkeypatch):
    """A module's frozen weights and scales do not send its calls through the dispatcher."""
    w, ws = (torch.nn.Parameter(t, requires_grad=False) for t in qz.quantize_weight(torch.randn(96, 256, device="cuda")))
    norm = torch.nn.Parameter(torch.ones(256, device="cuda"), requires_grad=False)
    x = torch.randn(5, 256, device="cuda")
    x8, xs, _ = qz.rms_norm(x, norm)
    want = qz.linear(x8, xs, w, ws)
    direct = []
    call = nat.call
    monkeypatch.setattr(nat, "call", lambda entry, *args: (direct.append(all(not isinstance(a, torch.Tensor) for a in args)), call(entry, *args)))
    monkeypatch.setattr(torch.ops, "fast_mimi_amd", None)  # the dispatcher's way
    assert torch.equal(qz.rms_norm(x, norm)[0].view(torch.uint8), x8.view(torch.uint8))
    assert torch.equal(qz.linear(x8, xs, w, ws), want) and direct == [True, True]
