"""Every kernel of the 8-bit products against 64 bits: ragged rows, outputs and inputs, each result type; how far
16-bit results are off in all, and scales at both ends."""

from __future__ import annotations

import pytest
import torch

import layer_ref as ref
from fast_mimi_amd import _native as nat
from fast_mimi_amd import quantized as qz
from training_ref import H, assert_within, half, step0

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def randn(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


def operands(m, n, k, spread=1.0):
    """Rows of very different size; values that spread around them by powers of two."""
    x = randn(m, k, seed=1) * torch.exp2((4 * randn(m, 1, seed=2)).round()) * torch.exp2((spread - 1) * randn(m, k, seed=3))
    w = randn(n, k, seed=4) * torch.exp2(randn(n, 1, seed=5).round()) * torch.exp2((spread - 1) * randn(n, k, seed=6))
    return *qz.quantize(x), *qz.quantize_weight(w)


def stand_for(values, scales, rows):
    return ref.stand_for(values, scales, rows).to(DEV)


def product(x, w, dtype):
    """(value, bound) of x [M, K] @ w [N, K]^T.  Of eight neighbouring products the 8-bit matrix instructions drop the
    bits that lie more than 2^-13 below the largest one's power of two; FP32 results are sums of exact products."""
    k = x.shape[1]
    y, size = x @ w.T, x.abs() @ w.abs().T
    bound = (k + 2) * H * size
    if dtype != F32:
        for first in range(0, k, 8):
            p = (x[:, None, first: first + 8] * w[None, :, first: first + 8]).abs()
            most = p.amax(2, keepdim=True)
            step = torch.exp2(torch.frexp(most)[1].double() - 14)  # frexp's mantissa is below 1
            bound += torch.where(most > 0, p - torch.floor(p / step) * step, 0.0).sum(2)
    return y, bound + half(dtype) * (y.abs() + bound) + step0(dtype)


def check(y, x, xs, w, ws, rows, columns, dtype):
    want, bound = product(stand_for(x[rows], xs[rows], 1), stand_for(w, ws, 128)[columns], dtype)
    got = y[rows][:, columns].double()
    fits = want.abs() + bound < torch.finfo(dtype).max  # what float16 cannot hold is an infinity there
    assert fits.double().mean() > 0.3
    assert_within("y", torch.where(fits, got, 0.0), torch.where(fits, want, 0.0), bound)


def some(n, tile):
    """The first and last of n, both sides of tiles' borders, and others."""
    borders = torch.arange(1, 4) * tile
    at = torch.cat((torch.arange(0, n, max(1, n // 9)), borders, borders - 1, torch.tensor([1, n - 1, n - 2, (n - 1) // tile * tile])))
    return torch.unique(at.clamp(0, n - 1)).to(DEV)


CASES = [(16, 333, 1040, "linear_rows_kernel<1>"), (32, 1000, 1008, "linear_rows_kernel<2>"),
         (65, 136, 2064, "linear_tile_kernel<64, 64> splits=2"), (40, 96, 8208, "linear_tile_kernel<64, 64> splits=8"),
         (65, 129, 4112, "linear_tile_kernel<64, 64> splits=4"), (300, 200, 144, "linear_tile_kernel<64, 64> splits=1"),
         (500, 4900, 272, "linear_tile_kernel<64, 128> splits=1"), (300, 8008, 1040, "linear_tile_kernel<64, 128> splits=1"),
         (1001, 6500, 144, "linear_tile_kernel<128, 128> splits=1"), (6500, 1040, 400, "linear_tile_kernel<128, 128> splits=1"),
         (4000, 3900, 400, "linear_tile_kernel<256, 256> splits=1"), (3999, 3904, 1168, "linear_tile_kernel<256, 256> splits=1"),
         (3841, 4001, 16, "linear_tile_kernel<256, 256> splits=1")]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n,k,plan", CASES)
def test_each_kernel(m, n, k, plan, dtype):
    """Some rows with all outputs, and some outputs with all rows."""
    assert nat.linear_fp8_plan(m, k, n) == plan
    x, xs, w, ws = operands(m, n, k)
    y = qz.linear(x, xs, w, ws, dtype)
    assert y.shape == (m, n) and y.dtype == dtype
    rows, columns = torch.arange(m, device=DEV), torch.arange(n, device=DEV)
    check(y, x, xs, w, ws, some(m, 64), columns, dtype)
    check(y, x, xs, w, ws, rows, some(n, 64), dtype)
    assert torch.equal(y, qz.linear(x, xs, w, ws, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n,k,plan", CASES)
def test_not_a_number_in_each_kernel(m, n, k, plan, dtype):
    """NaN values and scales reach their row's or columns' outputs and no others, also beside the last of either."""
    x, xs, w, ws = (t.view(torch.uint8).clone() for t in operands(m, n, k))
    f8, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    want = qz.linear(x.view(f8), xs.view(e8), w.view(f8), ws.view(e8), dtype)
    x[m - 1, k - 1], xs[m // 2, -1] = 127, 255
    nan = torch.zeros(m, n, dtype=torch.bool, device=DEV)
    nan[m - 1], nan[m // 2] = True, True
    rows = qz.linear(x.view(f8), xs.view(e8), w.view(f8), ws.view(e8), dtype)
    assert torch.equal(rows.isnan(), nan) and torch.equal(rows[~nan], want[~nan])
    x, xs, w, ws = (t.view(torch.uint8).clone() for t in operands(m, n, k))
    w[0, k - 1], ws[-1, 0] = 255, 255
    nan[:], nan[:, 0], nan[:, (n - 1) // 128 * 128:] = False, True, True
    columns = qz.linear(x.view(f8), xs.view(e8), w.view(f8), ws.view(e8), dtype)
    assert torch.equal(columns.isnan(), nan) and torch.equal(columns[~nan], want[~nan])


@pytest.mark.parametrize("values,figure", [("normal", 2e-5), ("positive", 2e-5), ("spread", 1e-4)])
@pytest.mark.parametrize("m,n,k", [(16, 2048, 128), (16, 2048, 8192), (300, 256, 128), (300, 256, 8192), (65, 512, 2064), (500, 4900, 1024),
                                   (1001, 6500, 1024), (4000, 3900, 1024)])
def test_how_far_16_bit_results_are_off(m, n, k, values, figure):
    """What the instructions drop is, in all, no more than documented of the results' size, at any number of inputs and also
    where every product has one sign.  (The root mean square of a sum of errors is at most the sum of theirs.)"""
    x, w = randn(m, k, seed=1), randn(n, k, seed=2) * k ** -0.5
    if values == "positive":
        x, w = x.abs(), w.abs()
    if values == "spread":
        x, w = x * torch.exp2(2 * randn(m, k, seed=3)), w * torch.exp2(2 * randn(n, k, seed=4))
    (x, xs), (w, ws) = qz.quantize(x), qz.quantize_weight(w)
    y = qz.linear(x, xs, w, ws, F16).double()
    want = stand_for(x, xs, 1) @ stand_for(w, ws, 128).T
    size = want.square().mean().sqrt()
    off, own = y - want, want.to(F16).double() - want
    assert off.square().mean().sqrt() <= own.square().mean().sqrt() + figure * size


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,n,k", [(5, 40, 256), (20, 40, 256), (300, 200, 2064), (500, 4900, 272)])
def test_scales_reach_far(m, n, k, dtype):
    """Both ends of the scales in the matrix instructions: their product decides."""
    x, w = randn(m, k, seed=1), randn(n, k, seed=2)
    (x, xs), (w, ws) = qz.quantize(x), qz.quantize_weight(w)
    plain = qz.linear(x, xs, w, ws, dtype)

    def moved(s, by):
        return (s.view(torch.uint8).int() + by).to(torch.uint8).view(torch.float8_e8m0fnu)

    for by in (100, -100):
        assert torch.equal(qz.linear(x, moved(xs, by), w, moved(ws, -by), dtype), plain)
    # FP32 results: within the range of a value times its scale.
    exact = qz.linear(x, xs, w, ws, F32)
    for by in (110, -110):
        assert torch.equal(qz.linear(x, moved(xs, by), w, moved(ws, -by), F32), exact)
    if dtype == BF16:
        for by in (60, -60):
            assert torch.equal(qz.linear(x, moved(xs, by), w, ws, dtype).double(), plain.double() * 2.0 ** by)
            assert torch.equal(qz.linear(x, xs, w, moved(ws, by), dtype).double(), plain.double() * 2.0 ** by)
