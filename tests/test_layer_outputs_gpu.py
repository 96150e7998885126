"""What the C entry points of the layer operators write, and what they leave: every output that is
given, and none that is not."""

from __future__ import annotations

import pytest
import torch

import layer_ref as ref
from fast_mimi_amd import _native as nat
from fast_mimi_amd import ops
from training_ref import assert_within

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = {F32: nat.DTYPE_F32, BF16: nat.DTYPE_BF16, F16: nat.DTYPE_F16}


# Channels of each row plan, of partial vectors, of rows read again at each step, and results past the L2.
@pytest.mark.parametrize("rows,c", [(3, 60), (5, 512), (33, 1000), (9, 2047), (3, 4096), (2, 8192), (2, 8200), (9000, 1024)])
@pytest.mark.parametrize("t,st", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)])
def test_rms_norm_gradients_that_are_given(rows, c, t, st):
    """dx is written at one type as at two, and may be left out; dresidual and dgamma have the same bits either way."""
    g = torch.Generator().manual_seed(c)
    x, r, dy, dh = (torch.randn(rows, c, generator=g).to(k).to(DEV) for k in (t, st, t, st))
    w = (1 + 0.1 * torch.randn(c, generator=g)).to(DEV)
    rstd = torch.rsqrt((x.double() + r.double()).square().mean(1) + 1e-5).float()
    size = nat.query("fm_rms_norm_backward_workspace_bytes", rows, c)
    ws = torch.empty(max(1, size // 4), device=DEV)

    def backward(dx):
        dr, dw = torch.full((rows, c), 77.0, dtype=st, device=DEV), torch.full((c,), 77.0, device=DEV)
        ops.call("fm_rms_norm_backward", dy, c, x, c, r, c, w, rstd, dh, c, rows, c, TYPES[t], TYPES[st], TYPES[F32], dx, dr, dw, ws, size)
        return dr, dw

    dx = torch.full((rows, c), 77.0, dtype=t, device=DEV)
    given, left = backward(dx), backward(None)
    assert all(torch.equal(a, b) for a, b in zip(given, left))
    if t == st:
        assert torch.equal(dx, given[0])
    few = slice(0, 200)
    val, err = ref.rms(x[few], r[few], w, dy[few], dh[few], 1e-5)
    assert_within("dx", dx[few], val["dx"], err["dx"])
    assert_within("dresidual", given[0][few], val["dresidual"], err["dresidual"])
