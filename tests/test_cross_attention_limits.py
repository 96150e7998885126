"""Cross attention at the ends of its documented range: 2097120 keys, and queries times heads per key head, over many
items or heads."""

from __future__ import annotations

import pytest
import torch

import layer_ref as ref
from fast_mimi_amd import _native as nat
from fast_mimi_amd import training as tr
from training_ref import assert_within

DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
MOST = 2_097_120


@pytest.mark.skipif(not nat.LIBRARY_PATH.is_file(), reason="library not built")
@pytest.mark.parametrize("batch,queries,keys", [(8192, 1, 600_000), (1 << 23, 1, MOST), (8192, MOST, 1), (2050, MOST, 2)])
def test_many_long_items_are_not_refused(batch, queries, keys):
    """Without an output the answer is that of a bad argument, not of an unsupported size."""
    P = 0x10000  # never dereferenced
    assert nat.library().fm_cross_attention_forward(P, 0, 8, 8, P, 0, 8, 8, P, 0, 8, 8, None, None, batch, queries, keys, 1, 1, 8, 0.25, 1,
                                                    None, P, None, 0, None) == 1000


def normal(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def check(q, k, v, grad, key_lengths=None, pick=None):
    kl = None if key_lengths is None else torch.tensor(key_lengths, dtype=torch.int32, device=DEV)
    out, lse = tr.cross_attention_forward(q, k, v, None, kl)
    got = {"out": out}
    if grad is not None:
        got.update(zip(("dq", "dk", "dv"), tr.cross_attention_backward(grad, q, k, v, out, lse, None, kl)))
    pick = range(q.shape[0]) if pick is None else pick
    for i in pick:
        part = slice(i, i + 1)
        val, err = ref.cross(q[part], k[part], v[part], q[part] if grad is None else grad[part], q.shape[3] ** -0.5,
                             None if key_lengths is None else key_lengths[part], None)
        for name, x in got.items():
            assert_within(name, x[part], val[name], err[name])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lengths", [None, [MOST - 1, 5]])
def test_the_most_keys(dtype, lengths):
    q, grad = (normal((2, 2, 1, 8), dtype, i) for i in range(2))
    k, v = (normal((2, MOST, 1, 8), dtype, i + 2) for i in range(2))
    check(q, k, v, grad, lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("h", [1, 8])
def test_the_most_rows(dtype, h):
    q, grad = (normal((1, MOST // h, h, 8), dtype, i) for i in range(2))
    k, v = (normal((1, 3, 1, 8), dtype, i + 2) for i in range(2))
    check(q, k, v, grad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("b,t,s,h,kv", [(70_001, 1, 3, 2, 1), (70_001, 5, 1, 1, 1), (300, 2, 2, 512, 256)])
def test_many_sequences(b, t, s, h, kv, dtype):
    q, grad = (normal((b, t, h, 16), dtype, i) for i in range(2))
    k, v = (normal((b, s, kv, 16), dtype, i + 2) for i in range(2))
    check(q, k, v, grad, None, [0, b // 3, b - 1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_items_over_shared_long_states(dtype):
    """4.9e9 keys in all, of one encoder for every item: read in place."""
    q = normal((8192, 1, 1, 8), dtype, 1)
    k, v = (normal((1, 600_000, 1, 8), dtype, i + 2).expand(8192, -1, -1, -1) for i in range(2))
    check(q, k, v, None, None, [0, 4095, 8191])
