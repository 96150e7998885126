"""RMS norm with the residual's addition and rotary positions on the GPU, against 64 bits."""

from __future__ import annotations

import pytest
import torch

import layer_ref as ref
from fast_mimi_amd import training as tr
from training_ref import H, SECOND_ORDER, assert_within

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def randn(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


# ----------------------------------------------------------------- RMS norm
@pytest.mark.parametrize("rows,c", [(1, 1), (3, 5), (2, 128), (33, 130), (7, 257), (5, 512), (19, 1000), (4, 2047), (9, 2048),
                                    (300, 64), (3, 4096), (2, 8191), (3, 8192), (2, 8200), (1, 20_001), (1100, 72)])
@pytest.mark.parametrize("types", [(F32, F32, F32), (BF16, BF16, BF16), (BF16, F32, F32), (F16, F16, F32), (F16, F32, F16)])
def test_rms_norm(rows, c, types):
    t, st, wt = types
    x, r = (0.5 * randn(rows, c, seed=1)).to(t).to(DEV), (2 * randn(rows, c, seed=2)).to(st).to(DEV)
    w, g = (1 + 0.1 * randn(c, seed=3)).to(wt).to(DEV), randn(rows, c, seed=4).to(t).to(DEV)
    gh = randn(rows, c, seed=5).to(st).to(DEV)
    val, err = ref.rms(x, r, w, g, gh, 1e-5)
    y, h, rstd = tr.rms_norm_forward(x, w, r)
    assert y.dtype == t and h.dtype == st and rstd.dtype == F32
    assert_within("y", y, val["y"], err["y"])
    assert_within("h", h, val["h"], err["h"])
    for parts in ((x, r),) + (((h, None),) if st == F32 else ()):
        dx, dr, dw = tr.rms_norm_backward(g, parts[0], rstd, w, parts[1], gh)
        assert dx.dtype == t and dr.dtype == st and dw.dtype == wt
        for name, got in (("dx", dx), ("dresidual", dr), ("dweight", dw)):
            assert_within(name, got, val[name], err[name])


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("weighted", [False, True])
def test_rms_norm_alone(t, weighted):
    """Without a residual, a stream's gradient or (also) a weight."""
    x, g = randn(37, 300, seed=1).to(t).to(DEV), randn(37, 300, seed=2).to(t).to(DEV)
    w = (1 + 0.1 * randn(300, seed=3)).to(t).to(DEV) if weighted else None
    val, err = ref.rms(x, None, w, g, None, 1e-6)
    y, h, rstd = tr.rms_norm_forward(x, w, eps=1e-6)
    assert h is x
    dx, dr, dw = tr.rms_norm_backward(g, x, rstd, w)
    assert dx is dr and (dw is None) == (not weighted)
    assert_within("y", y, val["y"], err["y"])
    assert_within("dx", dx, val["dx"], err["dx"])
    if weighted:
        assert_within("dweight", dw, val["dweight"], err["dweight"])


def test_rms_norm_of_strided_and_unaligned_rows():
    base, rbase = randn(40, 3 * 264, seed=1).to(BF16).to(DEV), randn(40, 2 * 301, seed=2).to(BF16).to(DEV)
    x, r = base[::2, 265: 265 + 259], rbase[1::2, 3: 3 + 259]
    w = randn(400, seed=3).to(BF16).to(DEV)[1: 260]
    g = randn(259, 20, seed=4).to(BF16).to(DEV).t()
    val, err = ref.rms(x, r, w, g, r, 1e-5)
    y, h, rstd = tr.rms_norm_forward(x, w, r)
    dx, dr, dw = tr.rms_norm_backward(g, x, rstd, w, r, r)
    for name, got in (("y", y), ("h", h), ("dx", dx), ("dresidual", dr), ("dweight", dw)):
        assert_within(name, got, val[name], err[name])


def test_rms_norm_empty_and_zero_rows():
    w = torch.ones(64, device=DEV)
    for shape in ((0, 64), (3, 0, 64)):
        x = torch.empty(shape, device=DEV)
        y, h, rstd = tr.rms_norm_forward(x, w, x)
        assert y.shape == h.shape == shape and rstd.shape == shape[:-1]
        dx, dr, dw = tr.rms_norm_backward(y, x, rstd, w, x)
        assert dx.shape == shape and not dw.any()
    x = torch.zeros(2, 64, device=DEV)
    y, h, rstd = tr.rms_norm_forward(x, w, x, 1e-5)
    assert not y.any() and not h.any() and torch.allclose(rstd, torch.full_like(rstd, 1e-5 ** -0.5))


def test_rms_norm_gradients_by_differences():
    """<dx, d> against the forward's central difference: what their distance may be follows from the outputs' bounds and
    from the same difference in 64 bits."""
    rows, c, step = 5, 200, 2.0 ** -5
    x, r, w, g, gh, d = (randn(rows, c, seed=i) for i in range(6))
    w = 1 + 0.1 * w[0]

    def loss(kernel, at):
        if kernel:
            y, h, _ = tr.rms_norm_forward(at.to(DEV), w.to(DEV), r.to(DEV))
            return (y.cpu().double() * g.double()).sum() + (h.cpu().double() * gh.double()).sum(), 0
        val, err = ref.rms(at, r, w, g, gh, 1e-5)
        return (val["y"] * g.double()).sum() + (val["h"] * gh.double()).sum(), \
            (err["y"] * g.abs().double()).sum() + (err["h"] * gh.abs().double()).sum()

    up, down = (x + step * d), (x - step * d)
    along = (up.double() - down.double()) / 2
    (ku, _), (kd, _), (eu, bu), (ed, bd) = loss(True, up), loss(True, down), loss(False, up), loss(False, down)
    val, err = ref.rms(x, r, w, g, gh, 1e-5)
    dx = tr.rms_norm_backward(g.to(DEV), x.to(DEV), tr.rms_norm_forward(x.to(DEV), w.to(DEV), r.to(DEV))[2], w.to(DEV),
                              r.to(DEV), gh.to(DEV))[0].cpu().double()
    curve = ((eu - ed) / 2 - (val["dx"] * along).sum()).abs()
    off = ((ku - kd) / 2 - (dx * along).sum()).abs()
    assert off <= SECOND_ORDER * ((bu + bd) / 2 + curve + (err["dx"] * along.abs()).sum())
    assert curve < 0.05 * (val["dx"] * along).sum().abs()  # the difference says something


def test_rms_norm_autograd():
    x, r, w = (randn(6, 96, seed=i).to(DEV).requires_grad_() for i in (1, 2, 3))
    w2 = w.detach()[0].clone().requires_grad_()
    y, h = tr.rms_norm(x, w2, r)
    gy, gh = randn(6, 96, seed=4).to(DEV), randn(6, 96, seed=5).to(DEV)
    for which in ((gy, gh), (gy, None), (None, gh)):
        outs = [(o, g) for o, g in zip((y, h), which) if g is not None]
        got = torch.autograd.grad([o for o, _ in outs], (x, w2, r), [g for _, g in outs], retain_graph=True, allow_unused=True)
        zero = torch.zeros_like(gy)
        val, err = ref.rms(x.detach(), r.detach(), w2.detach(), zero if which[0] is None else gy, which[1], 1e-5)
        for name, g in zip(("dx", "dweight", "dresidual"), got):
            assert_within(name, g, val[name], err[name])
    assert tr.rms_norm(x, w2).grad_fn is not None
    with torch.no_grad():
        assert torch.equal(tr.rms_norm(x, w2, r)[0], y)


@pytest.mark.parametrize("st", [BF16, F32])
def test_rms_norm_autograd_16_bits(st):
    x, r = randn(40, 136, seed=1).to(BF16).to(DEV).requires_grad_(), randn(40, 136, seed=2).to(st).to(DEV).requires_grad_()
    w = (1 + 0.1 * randn(136, seed=3)).to(DEV).requires_grad_()
    y, h = tr.rms_norm(x, w, r)
    gy, gh = randn(40, 136, seed=4).to(BF16).to(DEV), randn(40, 136, seed=5).to(st).to(DEV)
    got = torch.autograd.grad((y, h), (x, w, r), (gy, gh))
    val, err = ref.rms(x.detach(), r.detach(), w.detach(), gy, gh, 1e-5)
    for name, g in zip(("dx", "dweight", "dresidual"), got):
        assert_within(name, g, val[name], err[name])


# --------------------------------------------------------- rotary positions
FREQ = tr.rotary_frequencies


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,n,h,kv,d,rotated", [(1, 1, 1, 1, 2, 2), (2, 3, 4, 2, 64, 64), (1, 13, 8, 8, 64, 32), (3, 5, 3, 1, 80, 40),
                                                (2, 2, 2, 1, 13, 6), (1, 4, 2, 2, 96, 96), (2, 1, 5, 1, 20, 12), (1, 2, 1, 1, 512, 510),
                                                (1, 3, 2, 1, 7, 2), (2, 9, 20, 4, 128, 64)])
def test_rotary(t, interleaved, b, n, h, kv, d, rotated):
    packed = randn(b, n, (h + 2 * kv) * d, seed=1).to(t).to(DEV)
    q, k = packed[..., : h * d].view(b, n, h, d), packed[..., h * d: (h + kv) * d].view(b, n, kv, d)
    freq = FREQ(rotated, device=DEV)
    positions = torch.randint(0, 5000, (b, n), generator=torch.Generator().manual_seed(2))
    for inverse, call in ((False, tr.rotary_forward), (True, tr.rotary_backward)):
        got = call(q, k, freq, positions.to(DEV), interleaved, 1.25)
        for name, x, y in zip("qk", (q, k), got):
            want, bound = ref.rotary(x, freq.cpu(), positions, interleaved, 1.25, inverse)
            assert_within(name, y, want, bound)


@pytest.mark.parametrize("positions", [0, 7, -3, 1_000_000, 1 << 40, (1 << 53) - 4, -(1 << 53), torch.tensor([5, 0, 1 << 45, -9]),
                                       torch.tensor([3, 1, 2, 2_000_000_000], dtype=torch.int32)])
def test_rotary_positions(positions):
    """Far positions are as exact as near ones; no positions start at 0."""
    q = randn(2, 4, 3, 64, seed=3).to(DEV)
    freq = FREQ(64, device=DEV)
    given = positions.to(DEV) if isinstance(positions, torch.Tensor) else positions
    at = positions.long() if isinstance(positions, torch.Tensor) else torch.arange(4) + positions
    got, none = tr.rotary_forward(q, None, freq, given)
    want, bound = ref.rotary(q, freq.cpu(), at.expand(2, 4), False, 1.0)
    assert none is None
    assert_within("q", got, want, bound)
    if isinstance(positions, int) and positions == 0:
        assert torch.equal(got, tr.rotary_forward(q, None, freq)[0])


def test_rotary_strides_and_empty():
    x = randn(3, 6, 4, 64, seed=1).to(BF16).to(DEV)
    freq = FREQ(32, device=DEV)
    want = tr.rotary_forward(x, x, freq)
    for view in (x.transpose(0, 2).contiguous().transpose(0, 2), x.transpose(2, 3).contiguous().transpose(2, 3),
                 torch.cat((x[..., :1], x), -1)[..., 1:]):
        got = tr.rotary_forward(view, x, freq)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for shape in ((0, 6, 4, 64), (3, 0, 4, 64)):
        q, k = tr.rotary_forward(torch.empty(shape, device=DEV), torch.empty(shape, device=DEV), freq)
        assert q.shape == k.shape == shape
    q, k = tr.rotary_forward(x[:, :, :0], x, freq)
    assert q.shape == (3, 6, 0, 64) and torch.equal(k, want[1])


def test_rotary_keeps_infinities_of_other_channels():
    x = torch.full((1, 2, 1, 64), float("inf"), device=DEV)
    x[..., :32] = 1
    y = tr.rotary_forward(x, None, FREQ(32, device=DEV))[0]
    assert torch.isfinite(y[..., :32]).all() and torch.equal(y[..., 32:], x[..., 32:])


def test_rotary_autograd():
    """The gradient is the transposed rotation: against 64 bits, and <R x, g> = <x, R' g>."""
    q, k = randn(2, 5, 4, 64, seed=1).to(DEV).requires_grad_(), randn(2, 5, 2, 64, seed=2).to(DEV).requires_grad_()
    freq, positions = FREQ(48, device=DEV), torch.arange(10).view(2, 5) * 31
    gq, gk = randn(2, 5, 4, 64, seed=3).to(DEV), randn(2, 5, 2, 64, seed=4).to(DEV)
    for pos, at in ((positions.to(DEV), positions), (9, torch.arange(9, 14).expand(2, 5))):
        yq, yk = tr.rotary(q, k, freq, pos, True, 0.75)
        dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
        for name, got, g, x, y in (("dq", dq, gq, q, yq), ("dk", dk, gk, k, yk)):
            want, bound = ref.rotary(g, freq.cpu(), at, True, 0.75, True)
            assert_within(name, got, want, bound)
            a, b = (y.double() * g.double()).sum(), (x.double() * got.double()).sum()
            # Each output is off by at most 7 H of the pair's magnitudes.
            assert (a - b).abs() <= 14 * H * 2 * (x.double().abs().sum() * g.double().abs().max())
    (dq,) = torch.autograd.grad(tr.rotary(q, None, freq)[0], q, gq)
    assert torch.equal(dq, tr.rotary_backward(gq, None, freq)[0])


def test_rotary_scores_depend_on_distance():
    """What the rotation is for: products of turned queries and keys depend on their distance only."""
    q, k = randn(1, 1, 1, 64, seed=1).to(DEV), randn(1, 1, 1, 64, seed=2).to(DEV)
    freq = FREQ(64, device=DEV)
    scores = []
    for first in (0, 123, 1 << 33):
        a, b = tr.rotary_forward(q, None, freq, first + 11)[0], tr.rotary_forward(k, None, freq, first)[0]
        scores.append((a.double() * b.double()).sum().item())
    # Each factor is within 7 H of its pair's magnitudes, in each of 64 products.
    bound = 2 * 2 * 7 * H * (q.abs().double().sum() * k.abs().double().max()).item()
    assert max(scores) - min(scores) <= bound
