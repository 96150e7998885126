"""Keys that no query sees (a cache beyond the window, padding): their gradients are
zeros in blocks that have no rows at all, whatever the memory held before."""

from __future__ import annotations

import pytest
import torch

import training_ref as ref
from fast_mimi_amd import training as tr

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,t,s,h,kv,d,window", [
    (1, 40, 700, 4, 2, 128, 50), (60, 40, 700, 32, 16, 128, 50),  # both forms for heads of 128
    (1, 1, 300, 2, 2, 72, 1), (1, 40, 700, 4, 2, 64, 50), (100, 30, 300, 8, 8, 64, 7),
])
def test_unseen_keys_take_no_gradient(b, t, s, h, kv, d, window, dtype):
    g = torch.Generator().manual_seed(4)
    q, k, v, grad = (torch.randn(n, generator=g).to(dtype) for n in ((1, t, h, d), (1, s, kv, d), (1, s, kv, d), (1, t, h, d)))
    lengths = [s - t // 2] + [s] * (b - 1)
    many = [x.expand(b, -1, -1, -1).to(DEV) for x in (q, k, v, grad)]
    length = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    out, lse = tr.window_attention_forward(*many[:3], window, None, length)
    _, dk, dv = tr.window_attention_backward(many[3], *many[:3], out, lse, window, None, length)
    first = s - t - window + 1  # the first key that any query sees
    assert first > 32 and not dk[:, :first].any() and not dv[:, :first].any()
    for i in {0, b - 1}:
        want, bound = ref.attention(q, k, v, grad, window, d ** -0.5, [lengths[i]])
        ref.assert_within("dk", dk[i:i + 1], want["dk"], bound["dk"])
        ref.assert_within("dv", dv[i:i + 1], want["dv"], bound["dv"])
