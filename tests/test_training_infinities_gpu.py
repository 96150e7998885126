"""An infinite key that no row gives any probability: what it does to each gradient."""

from __future__ import annotations

import math

import pytest
import torch

from fast_mimi_amd import training as tr

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
def test_query_gradients_beside_an_infinite_key(dim, dtype):
    """Key 70 is -inf in channel 3 and scores -inf against every query.  It gets no
    gradient and changes no output; but dQ is dS times the keys, and 0 times -inf is
    NaN: channel 3 of the rows whose tile of 32 keys holds it (64 on), also of those
    before it, and nothing else."""
    g = torch.Generator().manual_seed(3)
    q, k, v, grad = (torch.randn(1, 100, 1, dim, generator=g).to(dtype).cuda() for _ in range(4))
    q = q.abs()
    low = k.clone()
    k[0, 70, 0, 3] = -math.inf
    low[0, 70, 0, 3] = -1000.0  # a score below -100 in base 2: its probability is lost beside any other
    q[..., 3] = q[..., 3] + 2
    out, lse = tr.window_attention_forward(q, k, v)
    dq, dk, dv = tr.window_attention_backward(grad, q, k, v, out, lse)
    out2, lse2 = tr.window_attention_forward(q, low, v)
    dq2, dk2, dv2 = tr.window_attention_backward(grad, q, low, v, out2, lse2)
    assert not dk[0, 70].any() and not dv[0, 70].any()
    assert torch.isfinite(out).all() and torch.isfinite(dk).all() and torch.isfinite(dv).all()
    nan = torch.zeros(dq.shape, dtype=torch.bool, device=dq.device)
    nan[0, 64:, 0, 3] = True
    assert torch.equal(dq.isnan(), nan)
    # FP32 blocks that meet the infinity run on other products: equal to FP32's own error only.
    tol = 1e-4 if dtype == torch.float32 else 0.0
    for a, b in ((out, out2), (dk, dk2), (dv, dv2), (dq.masked_fill(nan, 0), dq2.masked_fill(nan, 0))):
        rest = torch.arange(100, device=a.device) != 70
        assert (a - b)[:, rest].abs().max() <= tol
