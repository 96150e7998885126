"""Forms of the cross attention's kernels that only calls of many blocks take, against 64 bits."""

from __future__ import annotations

import pytest
import torch

import layer_ref as ref
from fast_mimi_amd import training as tr
from training_ref import assert_within

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("padded", [False, True])
# dK / dV by four waves with the keys in LDS (16 bits, more than 512 blocks); four and two waves of rows, and of keys.
@pytest.mark.parametrize("b,t,s,h,kv,d", [(5, 70, 840, 8, 8, 128), (17, 33, 500, 8, 4, 96), (6, 1000, 130, 8, 8, 128), (6, 130, 1000, 8, 8, 72),
                                          (4, 200, 300, 12, 12, 128), (12, 530, 140, 8, 8, 64), (12, 140, 530, 8, 8, 64), (8, 300, 270, 8, 8, 40)])
def test_many_blocks(b, t, s, h, kv, d, padded, dtype):
    g = torch.Generator().manual_seed(b)
    q, k, v, grad = (torch.randn(x, generator=g).to(dtype).to(DEV) for x in ((b, t, h, d), (b, s, kv, d), (b, s, kv, d), (b, t, h, d)))
    keys = [(s, 0, 1, s - 33, 31)[i % 5] for i in range(b)] if padded else None
    queries = [(t, t, t // 2, 0, t - 1, 33)[i % 6] for i in range(b)] if padded else None
    kl, ql = (None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV) for x in (keys, queries))
    out, lse = tr.cross_attention_forward(q, k, v, None, kl, ql)
    grads = tr.cross_attention_backward(grad, q, k, v, out, lse, None, kl, ql)
    val, err = ref.cross(q, k, v, grad, d ** -0.5, keys, queries)
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        assert_within(name, got, val[name], err[name])
