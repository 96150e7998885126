"""Attention of few queries over many keys: the forward cuts the keys over blocks
and joins the parts.  Out, the log-sum-exp and the gradients taken from it, against
the definition in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import training_ref as ref
from fast_mimi_amd import _native as nat
from fast_mimi_amd import training as tr

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def splits(b, t, s, h, kv, d, window):
    """How many parts the call has: its workspace holds a row of 64 or 128 columns
    and two statistics for each part and query head."""
    size = nat.library().fm_attention_forward_workspace_bytes(b, t, s, h, kv, d, s if window is None else window)
    return size // (4 * b * t * h * ((128 if d > 64 else 64) + 2))


def case(b, t, s, h, kv, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(n, generator=g).to(dtype) for n in ((b, t, h, d), (b, s, kv, d), (b, s, kv, d), (b, t, h, d))]


def check(parts, q, k, v, grad, window, lengths=None):
    b, t, h, d = q.shape
    assert splits(b, t, k.shape[1], h, k.shape[2], d, window) == parts
    want, bound = ref.attention(q, k, v, grad, window, d ** -0.5, lengths)
    # The hardware's exponential gives zero below 2^-126, so dS = P (dP - delta) is off by as much times dP - delta,
    # which is at most twice |G| |V|: a few 1e-37 of dK and dQ, where those are as small.
    size = 2 * grad.double().abs().sum(-1).amax() * v.double().abs().amax() * 2.0 ** -126 * d ** -0.5
    bound["dk"] = bound["dk"] + size * q.double().abs().sum(1).reshape(b, 1, k.shape[2], -1, d).sum(3)
    bound["dq"] = bound["dq"] + size * k.double().abs().sum(1).reshape(b, 1, k.shape[2], 1, d).expand(
        -1, -1, -1, h // k.shape[2], -1).reshape(b, 1, h, d)
    length = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    q, k, v, grad = (x.to(DEV) for x in (q, k, v, grad))
    out, lse = tr.window_attention_forward(q, k, v, window, None, length)
    grads = tr.window_attention_backward(grad, q, k, v, out, lse, window, None, length)
    for n, x in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        ref.assert_within(n, x, want[n], bound[n])
    return out, lse


def check_lse(lse, q, k, window, lengths=None):
    """log2 of the sum of exponentials; the scores' error is that of their products
    and of one FP32 rounding of a value of their size."""
    b, t, h, d = q.shape
    s, kv = k.shape[1], k.shape[2]
    for i in range(b):
        see = ref.visible(t, s, window, s if lengths is None else lengths[i])
        for a in range(h):
            Q, K = q[i, :, a].double(), k[i, :, a // (h // kv)].double()
            score = (Q @ K.T) * d ** -0.5 / math.log(2)
            want = (score * math.log(2)).masked_fill(~see, -torch.inf).logsumexp(1) / math.log(2)
            size = ((Q.abs() @ K.abs().T) * d ** -0.5 / math.log(2) * see).amax(1)
            got = lse[i, :, a].double().cpu()
            none = ~see.any(1)
            assert (got[none] == -torch.inf).all()
            off = (got - want)[~none].abs()
            assert (off <= ((d + 8) * ref.H * size + (s + 16) * ref.H * 1.5 + 2 * ref.H * want.abs())[~none]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("parts,b,t,s,h,kv,d,window", [
    (2, 1, 1, 897, 1, 1, 64, None),         # the fewest keys that are cut
    (2, 2, 2, 900, 4, 2, 64, None),
    (2, 1, 5, 1100, 6, 2, 72, None),        # nine tiles: five and four
    (2, 3, 1, 1100, 4, 4, 128, 1024),       # the window decides, and starts inside a tile
    (15, 2, 1, 8000, 8, 2, 64, None),       # 63 tiles in fives: the last two parts have none
    (15, 1, 5, 8000, 4, 1, 128, None),
    (10, 2, 2, 8000, 2, 2, 32, 5119),
    (64, 1, 1, 33000, 2, 1, 64, None),      # the most parts; 52 have keys
    (32, 16, 1, 16500, 1, 1, 8, None),      # the blocks' number decides
    (4, 1, 200, 2000, 1, 1, 64, None),      # several blocks of rows, each with its own tiles
    (3, 1, 70, 2000, 4, 2, 64, 1500),
])
def test_split_forward(parts, b, t, s, h, kv, d, window, dtype):
    q, k, v, grad = case(b, t, s, h, kv, d, dtype)
    _, lse = check(parts, q, k, v, grad, window)
    check_lse(lse, q, k, window)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("parts,t,s,window,lengths", [
    (2, 5, 1000, None, [1000, 996, 995, 0, 500, 999]),    # rows that are padding, clips that are nothing else
    (8, 40, 4000, None, [4000, 3970, 1, 3961, 3960, 128]),
    (2, 200, 2000, 1100, [2000, 1801, 1900, 1000]),
])
def test_split_forward_of_padded_clips(parts, t, s, window, lengths, dtype):
    q, k, v, grad = case(len(lengths), t, s, 4, 2, 64, dtype, 1)
    for i, n in enumerate(lengths):  # what padding holds reaches nothing
        q[i, max(0, n - (s - t)):], grad[i, max(0, n - (s - t)):], k[i, n:], v[i, n:] = 0, 0, 0, 0
    want = check(parts, q, k, v, grad, window, lengths)
    for i, n in enumerate(lengths):
        q[i, max(0, n - (s - t)):], grad[i, max(0, n - (s - t)):], k[i, n:], v[i, n:] = math.nan, math.inf, math.inf, math.nan
    length = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    out, lse = tr.window_attention_forward(q.to(DEV), k.to(DEV), v.to(DEV), window, None, length)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    check_lse(lse, q.nan_to_num(0, 0, 0), k.nan_to_num(0, 0, 0), window, lengths)


@pytest.mark.parametrize("dtype", TYPES)
def test_parts_of_very_different_sizes(dtype):
    """Scores that rise or fall by hundreds along the keys: most parts weigh nothing."""
    q, k, v, grad = case(1, 3, 2100, 2, 2, 64, dtype, 2)
    q = q.abs()
    for slope in (torch.linspace(-30, 30, 2100), torch.linspace(30, -30, 2100)):
        check(4, q, (k * 0.1 + slope[None, :, None, None]).to(dtype), v, grad, None)


def test_split_repeats_bit_for_bit_and_as_captured():
    q, k, v, _ = (x.to(DEV) for x in case(2, 1, 8000, 8, 2, 64, torch.float16, 3))
    first = tr.window_attention_forward(q, k, v)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = tr.window_attention_forward(q, k, v)
    for seed in (3, 4, 5):
        for to, fresh in zip((q, k, v), case(2, 1, 8000, 8, 2, 64, torch.float16, seed)):
            to.copy_(fresh)
        g.replay()
        again = tr.window_attention_forward(q, k, v)
        torch.cuda.synchronize()
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
        if seed == 3:
            assert torch.equal(out, first[0]) and torch.equal(lse, first[1])
