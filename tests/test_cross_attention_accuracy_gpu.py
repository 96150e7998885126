"""Which 16-bit gradients of cross attention are exact but for their rounding depends on an item's own lengths: not on
the batch around it, nor on whether its keys or rows are cut."""

from __future__ import annotations

import pytest
import torch

import layer_ref as ref
from fast_mimi_amd import _native as nat
from fast_mimi_amd import training as tr
from training_ref import assert_within

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16 = torch.bfloat16, torch.float16


def inputs(b, t, s, h, kv, d, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(shape, generator=g).to(dtype).to(DEV) for shape in ((b, t, h, d), (b, s, kv, d), (b, s, kv, d), (b, t, h, d))]


def check(args, names, pieces, key_lengths=None, query_lengths=None):
    q, k, v, grad = args
    kl, ql = (None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV) for x in (key_lengths, query_lengths))
    out, lse = tr.cross_attention_forward(q, k, v, None, kl, ql)
    grads = dict(zip(("dq", "dk", "dv"), tr.cross_attention_backward(grad, q, k, v, out, lse, None, kl, ql)))
    val, err = ref.cross(q, k, v, grad, q.shape[3] ** -0.5, key_lengths, query_lengths, pieces=pieces)
    for name in names.split():
        assert_within(name, grads[name], val[name], err[name])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("b,t,s,h,kv,d", [(40, 2, 300, 8, 4, 32), (9, 16, 130, 8, 2, 128), (70, 1, 33, 8, 8, 64), (3, 64, 512, 3, 3, 64)])
def test_items_in_larger_batches(b, t, s, h, kv, d, dtype):
    """Up to 64 rows a key head and 512 keys, whatever the batch."""
    check(inputs(b, t, s, h, kv, d, dtype), "dq dk dv", 2)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("t,h,kv,d,lengths", [(3, 2, 2, 64, [512, 200, 33]), (20, 2, 1, 128, [130, 0, 500]), (1, 4, 4, 64, [257, 31, 1])])
def test_cut_keys(t, h, kv, d, lengths, dtype):
    """Items whose keys are cut with those of longer ones beside them."""
    b, s = len(lengths) + 1, 3000
    assert nat.library().fm_cross_attention_backward_workspace_bytes(b, t, s, h, kv, d) > 0
    args = inputs(b, t, s, h, kv, d, dtype)
    check(args, "dk dv", 2, [s] + lengths)
    # The long one's dQ has the rounding of O in it.
    check(args, "dq", 1, [s] + lengths)
    check([x[1:] for x in args], "dq", 2, lengths)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("b,t,s,h,kv,d,lengths", [(9, 700, 64, 2, 2, 64, None), (1, 3000, 64, 2, 2, 64, None), (10, 500, 20, 8, 4, 128, None),
                                                  (3, 2500, 300, 2, 2, 64, [128, 1, 77]), (2, 1500, 400, 4, 2, 128, [64, 33])])
def test_few_keys_or_rows(b, t, s, h, kv, d, lengths, dtype):
    """dK and dV of up to 64 keys, or of up to 128 rows a key head, also where rows are cut."""
    check(inputs(b, t, s, h, kv, d, dtype), "dk dv", 2, None, lengths)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("b,t,s,h,kv,d", [(1, 65, 300, 2, 2, 64), (1, 64, 513, 2, 2, 64), (1, 3, 1500, 2, 2, 64), (1, 129, 65, 2, 2, 64),
                                          (2, 33, 513, 4, 2, 128), (1, 400, 65, 1, 1, 128)])
def test_beyond(b, t, s, h, kv, d, dtype):
    """Just above, and cut: within what the rounding of O, P and dS to 16 bits may add."""
    check(inputs(b, t, s, h, kv, d, dtype), "dq dk dv", 1)
