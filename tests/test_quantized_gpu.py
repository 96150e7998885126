"""Values, norms and products in 8 bits on the GPU, against 64 bits."""

from __future__ import annotations

import pytest
import torch

import layer_ref as ref
from fast_mimi_amd import quantized as qz
from fast_mimi_amd import training as tr
from training_ref import assert_within

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def randn(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def uneven(rows, c, seed, dtype):
    """Rows of very different size, a block of zeros, values at the borders of the format."""
    x = randn(rows, c, seed=seed) * torch.exp2(torch.randint(-12, 12, (rows, 1), generator=torch.Generator().manual_seed(seed)).float())
    x[0, : min(c, 128)] = 0
    if c > 5:
        x[-1, :6] = torch.tensor([448.0, -464.0, 17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10])
    return x.to(dtype)


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("rows,c", [(1, 1), (2, 16), (3, 127), (5, 128), (4, 129), (33, 257), (7, 1000), (300, 130), (2, 20_000)])
def test_quantize(t, rows, c):
    """The bits are the format's: the nearest value, ties to even, under the least power of two."""
    x = uneven(rows, c, 1, t)
    values, scales = qz.quantize(x.to(DEV))
    want, byte = ref.in_8_bits(x.double(), 1)
    assert values.dtype == torch.float8_e4m3fn and scales.dtype == torch.float8_e8m0fnu
    assert torch.equal(values.cpu().double(), want) and torch.equal(scales.cpu().view(torch.uint8).int(), byte.int())


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (130, 127), (257, 400), (64, 1024)])
def test_quantize_weight(t, n, k):
    w = uneven(n, k, 2, t)
    values, scales = qz.quantize_weight(w.to(DEV))
    want, byte = ref.in_8_bits(w.double(), 128)
    assert torch.equal(values.cpu().double(), want) and torch.equal(scales.cpu().view(torch.uint8).int(), byte.int())
    assert all(torch.equal(a.cpu().view(torch.uint8), b.cpu().view(torch.uint8))
               for a, b in zip(qz.quantize_weight(w.t().contiguous().t().to(DEV)), (values, scales)))


def test_quantize_limits():
    """The smallest and largest FP32 values; infinities and NaN make their own block NaN."""
    x = torch.zeros(6, 256)
    x[0, 3], x[1, 3], x[2, 3] = 2.0 ** -149, 2.0 ** -126, 3.4e38
    x[3, 200], x[4, 200], x[5, :] = float("inf"), float("nan"), 1.0
    x[3, 0] = x[4, 0] = 1.0
    values, scales = qz.quantize(x.to(DEV))
    got = ref.stand_for(values, scales, 1)
    # The first lies below what the smallest scale and the smallest value make; the others within half a step.
    assert (got[0] == 0).all() and got[1, 3] == 2.0 ** -126 and abs(got[2, 3] / 3.4e38 - 1) <= 2.0 ** -4
    assert torch.equal(scales.cpu().view(torch.uint8)[3:], torch.tensor([[119, 255], [119, 255], [119, 119]], dtype=torch.uint8))
    w, ws = qz.quantize_weight(torch.ones(16, 256, device=DEV))
    y = qz.linear(values, scales, w, ws, F32).cpu()
    assert y[3:5].isnan().all() and (y[5] == 256).all()


@pytest.mark.parametrize("rows,c", [(1, 4), (3, 64), (2, 128), (19, 200), (5, 512), (3, 1000), (4, 2047), (9, 2048), (2, 4096), (3, 8192),
                                    (2, 8200), (130, 136)])
@pytest.mark.parametrize("types", [(F32, F32, F32), (BF16, BF16, BF16), (BF16, F32, F32), (F16, F16, F32), (F16, F32, F16)])
def test_rms_norm(rows, c, types):
    t, st, wt = types
    x, r = (0.5 * randn(rows, c, seed=1)).to(t).to(DEV), (2 * randn(rows, c, seed=2)).to(st).to(DEV)
    w = (1 + 0.1 * randn(c, seed=3)).to(wt).to(DEV)
    values, scales, h = qz.rms_norm(x, w, r)
    assert torch.equal(h, tr.rms_norm_forward(x, w, r)[1])
    val, err = ref.rms(x, r, w, x, None, 1e-5)
    y, e = val["y"], err["y"] - ref.half(t) * val["y"].abs() - ref.step0(t)  # not rounded to t here
    # In e4m3: half a step is 2^-4 of a value, or 2^-10 of the scale.
    s = torch.exp2(scales.cpu().view(torch.uint8).double() - 127).repeat_interleave(128, 1)[:, :c]
    assert_within("y", ref.stand_for(values, scales, 1), y, e + torch.maximum(2.0 ** -4 * (y.abs() + e), 2.0 ** -10 * s))
    most = torch.nn.functional.pad(y.abs(), (0, -c % 128)).reshape(rows, -1, 128).amax(2)
    full = torch.exp2(scales.cpu().view(torch.uint8).double() - 127) * 448
    assert (most <= full * (1 + 1e-5)).all() and (most > full / 2 * (1 - 1e-5)).all()


def test_rms_norm_views_and_empty():
    x = randn(8, 300, seed=1).to(BF16).to(DEV)
    want = qz.rms_norm(x)
    assert want[2] is x
    wide = torch.zeros(8, 700, dtype=BF16, device=DEV)
    wide[:, 101:401] = x
    for a, b in zip(qz.rms_norm(wide[:, 101:401]), want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    values, scales, h = qz.rms_norm(x[:0], None, x[:0])
    assert values.shape == (0, 300) and scales.shape == (0, 3) and h.shape == (0, 300)
    assert qz.quantize(x[:0])[1].shape == (0, 3)


def operands(m, n, k, seed=1):
    x, xs = qz.quantize(uneven(m, k, seed, F32).to(DEV))
    w, ws = qz.quantize_weight((randn(n, k, seed=seed + 1) * torch.exp2(randn(n, 1, seed=seed + 2).round())).to(DEV))
    return x, xs, w, ws


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 32, 128), (1, 130, 400), (2, 64, 144), (5, 257, 1024), (16, 96, 256), (17, 128, 272),
                                   (33, 300, 640), (64, 128, 128), (65, 129, 2064), (100, 384, 512), (129, 257, 144), (300, 200, 384),
                                   (257, 520, 1040)])
def test_linear(m, n, k, dtype):
    x, xs, w, ws = operands(m, n, k)
    y = qz.linear(x, xs, w, ws, dtype)
    assert y.shape == (m, n) and y.dtype == dtype
    want, bound = ref.product(ref.stand_for(x, xs, 1), ref.stand_for(w, ws, 128), dtype)
    # What float16 cannot hold is an infinity there, as a rounding gives it.
    fits = want.abs() < torch.finfo(dtype).max
    assert_within("y", torch.where(fits, y.cpu().double(), 0.0), torch.where(fits, want, 0.0), bound)


def test_linear_shapes_and_views():
    x, xs, w, ws = operands(24, 96, 256)
    want = qz.linear(x, xs, w, ws)
    got = qz.linear(x.view(2, 3, 4, 256), xs.view(2, 3, 4, 2), w, ws)
    assert got.shape == (2, 3, 4, 96) and torch.equal(got.view(24, 96), want)
    assert torch.equal(qz.linear(x[3], xs[3], w, ws), want[3])
    wide = torch.zeros(24, 300, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    wide[:, 5:261] = x
    assert torch.equal(qz.linear(wide[:, 5:261], xs, w, ws), want)
    # Scales of a longer row, and of weights kept in another order.
    far = torch.full((24, 7), 255, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu)
    far.view(torch.uint8)[:, 3:5] = xs.view(torch.uint8)
    turned = ws.view(torch.uint8).t().contiguous().t().view(torch.float8_e8m0fnu)
    assert torch.equal(qz.linear(x, far[:, 3:5], w.view(torch.uint8).t().contiguous().t().view(torch.float8_e4m3fn), turned), want)
    assert qz.linear(x[:0], xs[:0], w, ws).shape == (0, 96)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n,k", [(3, 40, 256), (20, 300, 400), (90, 300, 1040), (300, 520, 256)])
def test_linear_of_not_a_number(m, n, k, dtype):
    """A NaN value or scale reaches its row's outputs, or its weights' columns, and no others."""
    x, xs, w, ws = operands(m, n, k)
    want = qz.linear(x, xs, w, ws, dtype)
    bad_x, bad_xs, bad_w, bad_ws = (t.view(torch.uint8).clone() for t in (x, xs, w, ws))
    bad_x[1, 200], bad_xs[m - 1, 0], bad_w[2, 5], bad_ws[-1, 1] = 127, 255, 255, 255
    nan = torch.zeros(m, n, dtype=torch.bool)
    nan[1], nan[m - 1] = True, True
    f8, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    rows = qz.linear(bad_x.view(f8), bad_xs.view(e8), w, ws, dtype)
    assert torch.equal(rows.isnan().cpu(), nan) and torch.equal(rows.cpu()[~nan], want.cpu()[~nan])
    nan[:], nan[:, 2], nan[:, (n - 1) // 128 * 128:] = False, True, True
    columns = qz.linear(x, xs, bad_w.view(f8), bad_ws.view(e8), dtype)
    assert torch.equal(columns.isnan().cpu(), nan) and torch.equal(columns.cpu()[~nan], want.cpu()[~nan])


def test_linear_scales_reach_far():
    """Scales of both ends: their products, not the partial ones, decide what is finite."""
    x, xs, w, ws = operands(20, 40, 256)
    plain = qz.linear(x, xs, w, ws, F32)
    for by in (60, -60):
        sx = (xs.view(torch.uint8).int() + by).to(torch.uint8).view(torch.float8_e8m0fnu)
        sw = (ws.view(torch.uint8).int() - by).to(torch.uint8).view(torch.float8_e8m0fnu)
        assert torch.equal(qz.linear(x, sx, w, sw, F32), plain)
        assert torch.equal(qz.linear(x, sx, w, ws, F32), plain * 2.0 ** by)


def test_gradients_are_refused():
    x = torch.ones(2, 128, device=DEV, requires_grad=True)
    for call in (lambda: qz.quantize(x), lambda: qz.quantize_weight(x), lambda: qz.rms_norm(x), lambda: qz.rms_norm(x.detach(), None, x)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
    with torch.no_grad():
        qz.rms_norm(x)
