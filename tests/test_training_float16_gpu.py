"""float16 attention where its operands would leave float16's range: small
probabilities, small and large gradients, against the definition in 64 bits.

P and dS are float16 operands of the second products.  They are held to half a
step relative to their own size, and to 2^-36 absolutely where they are small:
that stands in the place of float16's own smallest step (2^-24) in the bounds.
"""

from __future__ import annotations

import pytest
import torch

import training_ref as ref
from fast_mimi_amd import training as tr

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16 = torch.float16


def bounds(monkeypatch, *args):
    """``ref.attention`` with the operands' smallest step as above; the outputs'
    own is float16's."""
    own = ref.step0(F16)
    with monkeypatch.context() as m:
        m.setattr(ref, "step0", lambda t: 2.0 ** -36)
        val, err = ref.attention(*args)
    return val, {n: e + own for n, e in err.items()}


def run(q, k, v, grad, window=None, lengths=None):
    out, lse = tr.window_attention_forward(q, k, v, window, None, lengths)
    dq, dk, dv = tr.window_attention_backward(grad, q, k, v, out, lse, window, None, lengths)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def check(monkeypatch, batch, q, k, v, grad, window=None, names=("out", "dq", "dk", "dv")):
    """``batch`` copies of one clip (it decides how a block's waves share the
    work), the first and last against the definition."""
    val, err = bounds(monkeypatch, q, k, v, grad, window, q.shape[-1] ** -0.5, None)
    got = run(*(x.expand(batch, -1, -1, -1).to(DEV) for x in (q, k, v, grad)), window)
    for i in {0, batch - 1}:
        for n in names:
            # A gradient beyond the type's largest value rounds to infinity (key 0's, 3e6, below).
            over = val[n].abs() - ref.SECOND_ORDER * err[n] > torch.finfo(F16).max
            x = got[n][i:i + 1].double().cpu()
            assert torch.equal(x[over], val[n][over].sign() * torch.inf), n
            ref.assert_within(f"{n}[{i}]", x.masked_fill(over, 0.0), val[n].masked_fill(over, 0.0), err[n])


def axis(shape, values, at):
    """Zeros but for channel ``at``: ``values`` along the positions."""
    x = torch.zeros(shape)
    x[..., at] = values
    return x


@pytest.mark.parametrize("batch,queries,dim,heads", [(1, 300, 64, 1), (1, 100, 64, 1), (100, 300, 64, 1), (260, 300, 64, 1),
                                                     (1, 300, 128, 1), (64, 300, 128, 1), (1, 300, 32, 2)])
def test_small_probabilities_count(monkeypatch, batch, queries, dim, heads):
    """One key holds nearly all of the probability and its value is zero: what the
    511 others hold, 2^-21.6 each, is the output and the gradient of their values."""
    keys = 512
    q = axis((1, queries, heads, dim), 8.0, 0)
    b = 15.0 * (dim / 64) ** 0.5  # 21.6 bits of score above zero
    k = axis((1, keys, 1, dim), torch.where(torch.arange(keys) == 0, b, 0.0)[None, :, None], 0)
    v = torch.full((1, keys, 1, dim), 1000.0)
    v[:, 0] = 0.0
    grad = torch.full((1, queries, heads, dim), 1000.0)
    check(monkeypatch, batch, *(x.to(F16) for x in (q, k, v, grad)))


@pytest.mark.parametrize("keys,bits", [(1000, 23.7), (8000, 25.4), (30000, 26.7)])
def test_small_probabilities_of_a_token(keys, bits):
    """The same for one query over many keys (split over blocks from 1024 on)."""
    q, k = axis((1, 1, 1, 64), 8.0, 0).to(F16), axis((1, keys, 1, 64), 0.0, 0)
    k[:, 0, 0, 0] = bits / 1.44269504
    k = k.to(F16)
    v = torch.full((1, keys, 1, 64), 60000.0, dtype=F16)
    v[:, 0] = 0
    out, lse = tr.window_attention_forward(q.to(DEV), k.to(DEV), v.to(DEV))
    p = torch.exp(-k[0, 0, 0, 0].double())  # of each other key against the first one
    total = 1 + (keys - 1) * p
    want = (keys - 1) * 60000.0 * p / total
    # Half a step of 2^-35 of the largest for each, the score's exponential and the sums in FP32, the result's rounding.
    bound = (keys * 60000.0 * 2.0 ** -36 + want * ((keys + 200) * ref.H + ref.half(F16))) * 1.01
    assert (out.double().cpu() - want).abs().max() <= bound
    assert abs(lse.item() - (k[0, 0, 0, 0].item() * 1.4426950408889634 + torch.log2(total).item())) <= 1e-5


@pytest.mark.parametrize("batch,dim,heads", [(1, 64, 1), (20, 64, 1), (100, 64, 1), (1, 128, 1), (40, 128, 2), (1, 32, 4)])
@pytest.mark.parametrize("size", [1e-5, 1e-3, 1.0])
def test_gradients_of_any_size(monkeypatch, batch, dim, heads, size):
    """Equal scores over 500 keys whose values are one or minus one: every dS of a
    full row has the same magnitude, 64 size / 500, so their roundings add up."""
    n = 1000
    sign = 1.0 - 2.0 * (torch.arange(n) % 2)
    q = axis((1, n, heads, dim), 64.0, 1)
    k = axis((1, n, 1, dim), 8.0 * sign[None, :, None], 0) + axis((1, n, 1, dim), 1.0, 1)
    v = sign[None, :, None, None].expand(1, n, 1, dim)
    grad = torch.full((1, n, heads, dim), size)
    check(monkeypatch, batch, *(x.to(F16) for x in (q, k, v, grad)), 500)


@pytest.mark.parametrize("batch,dim", [(1, 64), (100, 64), (1, 128), (40, 128)])
def test_products_beyond_float16(monkeypatch, batch, dim):
    """P (dP - delta) of 3e5 and more, where the gradients themselves are float16."""
    n = 600
    sign = 1.0 - 2.0 * (torch.arange(n) % 2)
    q = axis((1, n, 1, dim), 2.0 ** -10, 1)
    k = axis((1, n, 1, dim), 2.0 ** -7 * sign[None, :, None], 0) + axis((1, n, 1, dim), 1.0, 1)
    v = (500.0 * sign)[None, :, None, None].expand(1, n, 1, dim)
    grad = torch.full((1, n, 1, dim), 1000.0)
    check(monkeypatch, batch, *(x.to(F16) for x in (q, k, v, grad)), 100)


@pytest.mark.parametrize("t,s,heads,kv,dim,window", [(200, 200, 4, 2, 64, None), (400, 400, 1, 1, 128, 150), (20, 300, 4, 2, 72, None),
                                                     (130, 130, 2, 2, 32, 40)])
@pytest.mark.parametrize("rising", [True, False])
def test_rows_of_very_different_sizes(t, s, heads, kv, dim, window, rising):
    """Gradients from 1e-6 to 1e3 over the rows, and values that grow along the
    keys: the operands' levels fall on the way through a row's keys and a key's rows."""
    g = torch.Generator().manual_seed(5)
    q, grad = (torch.randn(2, t, heads, dim, generator=g) for _ in range(2))
    k, v = (torch.randn(2, s, kv, dim, generator=g) for _ in range(2))
    rows, cols = torch.logspace(-6, 3, t), torch.logspace(-3, 1, s)
    rows, cols = (rows, cols) if rising else (rows.flip(0), cols.flip(0))
    q, k, v, grad = (x.to(F16) for x in (q, k, v * cols[None, :, None, None], grad * rows[None, :, None, None]))
    val, err = ref.attention(q, k, v, grad, window, dim ** -0.5, None)
    for n, x in run(*(x.to(DEV) for x in (q, k, v, grad)), window).items():
        ref.assert_within(n, x, val[n], err[n])


def test_an_infinite_gradient_stays_with_its_row():
    """dQ of the other rows of its tile is as without it."""
    g = torch.Generator().manual_seed(6)
    q, k, v, grad = (torch.randn(1, 100, 1, 64, generator=g).to(F16).to(DEV) for _ in range(4))
    clean = run(q, k, v, grad)
    grad[0, 40, 0, 3] = torch.inf
    got = run(q, k, v, grad)
    others = torch.arange(100) != 40
    assert torch.equal(got["dq"][:, others], clean["dq"][:, others])
    assert torch.equal(got["out"], clean["out"])
