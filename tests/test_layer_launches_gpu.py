"""Calls that take more than one launch, or a second form of a kernel: the rows behind a launch's most, and parts of cut
walks whose values want FP32 products."""

from __future__ import annotations

import pytest
import torch

import layer_ref as ref
from fast_mimi_amd import _native as nat
from fast_mimi_amd import quantized as qz
from fast_mimi_amd import training as tr
from training_ref import assert_within

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def randn(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


def same(a, b):
    return torch.equal(a.view(torch.uint8) if a.element_size() == 1 else a, b.view(torch.uint8) if b.element_size() == 1 else b)


@pytest.mark.parametrize("t,st", [(F32, F32), (BF16, BF16), (BF16, F32)])
def test_norms_of_many_rows(t, st):
    """2^23 rows are a launch's most."""
    rows, c, first = (1 << 23) + 1003, 12, (1 << 23) - 500
    x, r, w, g = randn(rows, c, seed=1).to(t), randn(rows, c, seed=2).to(st), randn(c, seed=3).to(t), randn(rows, c, seed=4).to(t)
    tail = slice(first, rows)
    y, h, rstd = tr.rms_norm_forward(x, w, r)
    assert all(same(a[tail], b) for a, b in zip((y, h, rstd), tr.rms_norm_forward(x[tail], w, r[tail])))
    dx, dr, _ = tr.rms_norm_backward(g, x, rstd, w, r)
    assert all(same(a[tail], b) for a, b in zip((dx, dr), tr.rms_norm_backward(g[tail], x[tail], rstd[tail], w, r[tail])))
    got = qz.rms_norm(x, w, r)
    assert all(same(a[tail], b) for a, b in zip(got, qz.rms_norm(x[tail], w, r[tail])))
    val, err = ref.rms(x[-100:], r[-100:], w, g[-100:], None, 1e-5)
    for name, a in (("y", y), ("h", h), ("dx", dx), ("dresidual", dr)):
        assert_within(name, a[-100:], val[name], err[name])


def test_quantized_rows_of_two_launches():
    """2^30 vectors are a launch's most: 2^26 rows of one block of bfloat16."""
    rows = (1 << 26) + 77
    x = randn(rows, 2, seed=1).to(BF16)
    values, scales = qz.quantize(x)
    for part in (slice(0, 300), slice((1 << 26) - 300, rows)):
        want, byte = ref.in_8_bits(x[part].double().cpu(), 1)
        assert torch.equal(values[part].cpu().double(), want) and torch.equal(scales[part].cpu().view(torch.uint8).int(), byte.int())


def test_a_rotation_of_two_launches():
    """2^24 blocks are a launch's most: here one position of two heads each."""
    n, h, d = 540, 65_534, 512
    q = randn(1, n, 1, d, seed=1).to(BF16).expand(1, n, h, d)
    freq = tr.rotary_frequencies(510, device=DEV)
    got, _ = tr.rotary_forward(q, None, freq, 3)
    want, bound = ref.rotary(q[:, :, :1], freq.cpu(), (torch.arange(n) + 3)[None], False, 1.0)
    for at in (0, h // 2, h - 1):
        assert_within("q", got[:, :, at: at + 1], want, bound)


@pytest.mark.parametrize("b,t,s,h,kv,d", [(1, 3, 1500, 2, 2, 64), (1, 1400, 5, 2, 2, 64), (1, 2600, 33, 1, 1, 32)])
def test_large_values_in_some_parts(b, t, s, h, kv, d):
    """Parts that meet values beyond 2^36 run on FP32 products, the others on pieces, and are joined alike."""
    assert nat.library().fm_cross_attention_backward_workspace_bytes(b, t, s, h, kv, d) > 0
    q, k, v, grad = randn(b, t, h, d, seed=1), randn(b, s, kv, d, seed=2), randn(b, s, kv, d, seed=3), randn(b, t, h, d, seed=4)
    far = torch.ones(s, device=DEV)
    far[s // 2:] = 2.0 ** 45
    v = v * far[None, :, None, None]
    rows = torch.ones(t, device=DEV)
    rows[t // 3:] = 2.0 ** 40
    grad = grad * rows[None, :, None, None]
    out, lse = tr.cross_attention_forward(q, k, v)
    grads = tr.cross_attention_backward(grad, q, k, v, out, lse)
    val, err = ref.cross(q, k, v, grad, d ** -0.5, None, None)
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        assert_within(name, got, val[name], err[name])
