"""Attention to another sequence on the GPU, forward and backward, against 64 bits."""

from __future__ import annotations

import pytest
import torch

import layer_ref as ref
from fast_mimi_amd import training as tr
from training_ref import SECOND_ORDER, assert_within

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def inputs(b, t, s, h, kv, d, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    q, k, v, grad = (torch.randn(shape, generator=g).to(dtype).to(DEV) for shape in
                     ((b, t, h, d), (b, s, kv, d), (b, s, kv, d), (b, t, h, d)))
    return q, k, v, grad


def check(q, k, v, grad, scale=None, key_lengths=None, query_lengths=None):
    kl, ql = (None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV) for x in (key_lengths, query_lengths))
    out, lse = tr.cross_attention_forward(q, k, v, scale, kl, ql)
    grads = tr.cross_attention_backward(grad, q, k, v, out, lse, scale, kl, ql)
    val, err = ref.cross(q, k, v, grad, q.shape[3] ** -0.5 if scale is None else scale, key_lengths, query_lengths)
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        assert got.dtype == q.dtype and got.is_contiguous()
        assert_within(name, got, val[name], err[name])
    return out, lse, grads


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("b,t,s,h,kv,d", [(1, 1, 1, 1, 1, 64), (2, 13, 7, 2, 2, 64), (1, 7, 130, 4, 2, 32), (2, 33, 31, 2, 1, 128),
                                          (1, 100, 3, 3, 3, 16), (1, 65, 257, 2, 2, 80), (3, 1, 40, 8, 2, 64), (2, 129, 129, 6, 2, 96),
                                          (1, 300, 20, 1, 1, 120)])
def test_cross_attention(b, t, s, h, kv, d, dtype):
    check(*inputs(b, t, s, h, kv, d, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
def test_padding(d, dtype):
    """Lengths of every kind; what padding holds reaches nothing."""
    b, t, s = 7, 70, 150
    keys, queries = [150, 1, 0, 33, 149, 200, -5], [70, 70, 70, 1, 0, 33, 64]
    q, k, v, grad = inputs(b, t, s, 4, 2, d, dtype)
    first = check(q, k, v, grad, None, keys, queries)
    for i in range(b):
        rows, n = max(0, min(queries[i], t)), max(0, min(keys[i], s))
        q[i, rows:], grad[i, rows:], k[i, n:], v[i, n:] = float("nan"), float("inf"), float("inf"), float("nan")
    kl, ql = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (keys, queries))
    out, lse = tr.cross_attention_forward(q, k, v, None, kl, ql)
    grads = tr.cross_attention_backward(grad, q, k, v, out, lse, None, kl, ql)
    assert torch.equal(out, first[0]) and torch.equal(lse, first[1])
    assert all(torch.equal(a, c) for a, c in zip(grads, first[2]))
    assert (lse[2] == -torch.inf).all() and not out[2].any() and not grads[0][6].any()
    assert (lse[3, 1:] == -torch.inf).all() and not out[3, 1:].any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("b,t,s,h,kv,d", [(1, 3, 1500, 2, 1, 64), (2, 40, 1300, 1, 1, 128), (1, 1, 2600, 4, 4, 64)])
def test_long_keys_are_cut(b, t, s, h, kv, d, dtype):
    """Few rows over many keys: the forward's and dQ's keys are split over blocks."""
    from fast_mimi_amd import _native as nat

    assert nat.library().fm_cross_attention_forward_workspace_bytes(b, t, s, h, kv, d) > 0
    assert nat.library().fm_cross_attention_backward_workspace_bytes(b, t, s, h, kv, d) > 0
    q, k, v, grad = inputs(b, t, s, h, kv, d, dtype)
    check(q, k, v, grad)
    check(q, k, v, grad, 0.3, [s - 700 * i - 129 for i in range(b)], [max(1, t - 1)] * b)
    check(q, k, v, grad, 0.3, [5 * i for i in range(b)])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("b,t,s,h,kv,d", [(1, 1400, 5, 2, 2, 64), (2, 700, 40, 2, 1, 128), (1, 2600, 33, 1, 1, 32)])
def test_long_queries_are_cut(b, t, s, h, kv, d, dtype):
    """Many rows over few keys: dK's and dV's rows are split over blocks."""
    from fast_mimi_amd import _native as nat

    assert nat.library().fm_cross_attention_backward_workspace_bytes(b, t, s, h, kv, d) > 0
    q, k, v, grad = inputs(b, t, s, h, kv, d, dtype)
    check(q, k, v, grad)
    check(q, k, v, grad, 0.3, [s - i for i in range(b)], [t - 301 * (i + 1) for i in range(b)])
    check(q, k, v, grad, None, None, [7 + 100 * i for i in range(b)])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("b,t,s,h,kv,d", [(4, 1540, 510, 8, 8, 32), (4, 2309, 300, 8, 8, 64)])
def test_middling_blocks_are_cut(b, t, s, h, kv, d, dtype):
    """Blocks for one round, not two, and a long walk: dK's and dV's rows are split over blocks of more waves."""
    from fast_mimi_amd import _native as nat

    assert nat.library().fm_cross_attention_backward_workspace_bytes(b, t, s, h, kv, d) > 0
    q, k, v, grad = inputs(b, t, s, h, kv, d, dtype)
    check(q, k, v, grad)
    check(q, k, v, grad, 0.3, [s, 0, 1, s - 33], [t, t, 770, 0])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("b,t,s,h,kv,d,names", [(1, 1, 33, 2, 2, 64, "dq dk dv"), (1, 4, 64, 2, 1, 64, "dq dk dv"), (3, 2, 300, 4, 4, 32, "dq dk dv"),
                                                (2, 30, 130, 4, 2, 128, "dq dk dv"), (1, 129, 2, 2, 2, 64, "dk dv"), (2, 700, 5, 2, 1, 128, "dk dv"),
                                                (1, 3000, 33, 2, 2, 64, "dk dv")])
def test_few_results_are_exact(b, t, s, h, kv, d, names, dtype):
    """Gradients of few rows or keys in all, where chance would add to a rounding within them: only their own shows."""
    q, k, v, grad = inputs(b, t, s, h, kv, d, dtype)
    out, lse = tr.cross_attention_forward(q, k, v)
    grads = dict(zip(("dq", "dk", "dv"), tr.cross_attention_backward(grad, q, k, v, out, lse)))
    val, err = ref.cross(q, k, v, grad, d ** -0.5, None, None, pieces=2)
    for name in names.split():
        assert_within(name, grads[name], val[name], err[name])


def test_views():
    """Slices of packed projections, transposed heads, odd offsets."""
    g = torch.Generator().manual_seed(3)
    kv = torch.randn(2, 50, 2 * 2 * 64, generator=g).to(BF16).to(DEV)
    k, v = kv[..., :128].view(2, 50, 2, 64), kv[..., 128:].view(2, 50, 2, 64)
    q = torch.randn(2, 4, 33, 64, generator=g).to(BF16).to(DEV).transpose(1, 2)
    grad = torch.randn(2, 33, 4, 65, generator=g).to(BF16).to(DEV)[..., 1:]
    out, lse, grads = check(q, k, v, grad)
    again = tr.cross_attention_forward(*(x.contiguous() for x in (q, k, v)))
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    shared = k[:1].expand(2, -1, -1, -1)
    check(q, shared, v, grad)


def test_empty():
    for b, t, s in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k, v, grad = inputs(b, t, s, 2, 2, 64, BF16)
        out, lse = tr.cross_attention_forward(q, k, v)
        grads = tr.cross_attention_backward(grad, q, k, v, out, lse)
        assert out.shape == q.shape and not out.any() and (lse == -torch.inf).all()
        assert [x.shape for x in grads] == [x.shape for x in (q, k, v)] and not any(x.any() for x in grads)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_large_scores(dtype):
    """One key takes all of a row; scores in the thousands."""
    q, k, v, grad = inputs(1, 40, 60, 2, 2, 64, dtype)
    check(20 * q, 20 * k, v, grad)


def test_large_values_in_fp32():
    """Magnitudes beyond what three 16-bit pieces hold run on FP32 products."""
    q, k, v, grad = inputs(1, 40, 60, 1, 1, 64, F32)
    check(q, k, v * 2.0 ** 50, grad)
    check(q * 2.0 ** -40, k * 2.0 ** 40, v, grad)


def test_the_same_call_gives_the_same_bits():
    args = inputs(1, 1400, 40, 4, 2, 64, BF16)
    first = check(*args)
    again = check(*args)
    assert all(torch.equal(a, b) for a, b in zip((*first[:2], *first[2]), (*again[:2], *again[2])))


def test_agrees_with_window_attention_where_the_mask_hides_nothing():
    """One query at the last position of its keys sees them all in either form, each within its
    bound of the exact result (the sums run in orders of their own)."""
    q, k, v, grad = inputs(3, 1, 40, 4, 2, 64, BF16)
    _, err = ref.cross(q, k, v, grad, 64 ** -0.5, None, None)
    assert_within("out", tr.cross_attention(q, k, v), tr.window_attention(q, k, v), 2 * err["out"])


def test_autograd_and_differences():
    q, k, v, grad = (x.requires_grad_() for x in inputs(2, 12, 20, 4, 2, 32, F32))
    kl = torch.tensor([20, 9], dtype=torch.int32, device=DEV)
    out = tr.cross_attention(q, k, v, None, kl)
    got = torch.autograd.grad(out, (q, k, v), grad.detach())
    args = [x.detach() for x in (q, k, v, grad)]
    val, err = ref.cross(*args, 32 ** -0.5, [20, 9], None)
    step = 2.0 ** -6
    for i, name in enumerate(("dq", "dk", "dv")):
        assert_within(name, got[i], val[name], err[name])
        # Along a random direction: what the kernel's central difference may be off by follows from the
        # outputs' bounds, and from the same difference in 64 bits.
        d = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i)).to(DEV)
        sides = []
        for sign in (1, -1):
            at = list(args)
            at[i] = args[i] + sign * step * d
            want, bound = ref.cross(*at, 32 ** -0.5, [20, 9], None)
            g = grad.detach().double().cpu()
            sides.append((at[i].double().cpu(), (tr.cross_attention(*at[:3], None, kl).double().cpu() * g).sum(),
                          (want["out"] * g).sum(), (bound["out"] * g.abs()).sum()))
        (up, ku, eu, bu), (down, kd, ed, bd) = sides
        along = (up - down) / 2
        curve = ((eu - ed) / 2 - (val[name] * along).sum()).abs()
        off = ((ku - kd) / 2 - (got[i].double().cpu() * along).sum()).abs()
        assert off <= SECOND_ORDER * ((bu + bd) / 2 + curve + (err[name] * along.abs()).sum())
        assert curve < 0.05 * ((val[name] * along).sum().abs() + 1e-3 * (val[name] * along).abs().sum())
