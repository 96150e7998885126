"""Norms and rotations whose results go past the L2 cache, against 64 bits at both ends and in between."""

from __future__ import annotations

import pytest
import torch

import layer_ref as ref
from fast_mimi_amd import training as tr
from training_ref import assert_within

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def randn(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


@pytest.mark.parametrize("rows,c", [(180_000, 257), (90_001, 512), (45_000, 1000), (22_000, 2047), (11_000, 4096), (5600, 8192)])
@pytest.mark.parametrize("types", [(F32, F32, F32), (BF16, BF16, BF16), (BF16, F32, F32), (F16, F32, F16)])
def test_rms_norm(rows, c, types):
    t, st, wt = types
    x, r, w = (0.5 * randn(rows, c, seed=1)).to(t), (2 * randn(rows, c, seed=2)).to(st), (1 + 0.1 * randn(c, seed=3)).to(wt)
    g, gh = randn(rows, c, seed=4).to(t), randn(rows, c, seed=5).to(st)
    y, h, rstd = tr.rms_norm_forward(x, w, r)
    dx, dr, dw = tr.rms_norm_backward(g, x, rstd, w, r, gh)
    for part in (slice(0, 40), slice(rows // 2 - 20, rows // 2 + 20), slice(rows - 40, rows)):
        val, err = ref.rms(x[part], r[part], w, g[part], gh[part], 1e-5)
        for name, got in (("y", y), ("h", h), ("dx", dx), ("dresidual", dr)):
            assert_within(name, got[part], val[name], err[name])
    # All rows at once, in 64 bits: the sum over them, whose FP32 additions are rows deep at most.
    want, bound = torch.zeros(c, dtype=torch.float64, device=DEV), torch.zeros(c, dtype=torch.float64, device=DEV)
    for first in range(0, rows, 20_000):
        part = slice(first, first + 20_000)
        s = x[part].double() + r[part].double()
        hh = g[part].double() * s / torch.sqrt(s.square().mean(1, keepdim=True) + 1e-5)
        want += hh.sum(0)
        bound += hh.abs().sum(0)
    # A product carries the row's sum (c / 16 + 20 roundings, as in layer_ref) and its own; partial sums are joined from 512
    # to 1024 blocks, so a column's chain has no more additions than rows.
    assert_within("dweight", dw, want.cpu(), ((rows + c / 16 + 20) * ref.H * bound + ref.half(wt) * want.abs()).cpu() + ref.step0(wt))


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,n,h,kv,d,rotated", [(8, 4095, 16, 4, 128, 128), (8, 4095, 16, 4, 128, 64), (3, 9000, 16, 8, 160, 96), (5, 7001, 20, 4, 96, 64)])
def test_rotary(b, n, h, kv, d, rotated, interleaved, t):
    packed = randn(b, n, (h + kv) * d, seed=1).to(t)
    q, k = packed[..., : h * d].view(b, n, h, d), packed[..., h * d:].view(b, n, kv, d)
    freq = tr.rotary_frequencies(rotated, device=DEV)
    got = tr.rotary_forward(q, k, freq, 5, interleaved, 1.25)
    some = torch.tensor([0, 1, n // 2, n - 2, n - 1])
    for name, x, y in zip("qk", (q, k), got):
        want, bound = ref.rotary(x[:, some], freq.cpu(), (some + 5).expand(b, -1), interleaved, 1.25)
        assert_within(name, y[:, some], want, bound)
    # Every other position: as a call of its own, whose results stay in the caches, gives it.
    assert b * n * (h + kv) * d * q.element_size() >= 128 << 20
    for first in range(0, n, 1000):
        part = slice(first, min(n, first + 1000))
        for a, c in zip(got, tr.rotary_forward(q[:, part], k[:, part], freq, 5 + first, interleaved, 1.25)):
            assert torch.equal(a[:, part], c)
