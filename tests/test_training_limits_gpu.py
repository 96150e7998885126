"""The training operators at the ends of their documented ranges: the most keys and
rows, the most sequences, every head width, wide and single embedding columns."""

from __future__ import annotations

import pytest
import torch

import training_ref as ref
from fast_mimi_amd import training as tr

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
MOST = 2_097_120


def normal(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def run(q, k, v, grad, window):
    out, lse = tr.window_attention_forward(q, k, v, window)
    return {"out": out, **dict(zip(("dq", "dk", "dv"), tr.window_attention_backward(grad, q, k, v, out, lse, window)))}


@pytest.mark.parametrize("dtype", TYPES)
def test_the_most_positions(dtype):
    """2097120 positions under a window: parts of the sequence against the definition.
    A row's keys and a key's rows are within 32, so a part's inside is as in the whole."""
    window = 33
    q, k, v, grad = (normal((1, MOST, 1, 8), dtype, i) for i in range(4))
    got = run(q, k, v, grad, window)
    for first in (0, 1_000_001, MOST - 300):
        part = [x[:, first:first + 300] for x in (q, k, v, grad)]
        want, bound = ref.attention(*part, window, 8 ** -0.5, None)
        lo = 0 if first == 0 else window
        hi = 300 if first + 300 == MOST else 300 - window
        for n, x in got.items():
            ref.assert_within(n, x[:, first + lo:first + hi], want[n][:, lo:hi], bound[n][:, lo:hi])


@pytest.mark.parametrize("dtype", TYPES)
def test_two_queries_over_the_most_keys(dtype):
    q, grad = (normal((1, 2, 1, 8), dtype, i) for i in range(2))
    k, v = (normal((1, MOST, 1, 8), dtype, i + 2) for i in range(2))
    want, bound = ref.attention(q, k, v, grad, None, 8 ** -0.5, None)
    for n, x in run(q, k, v, grad, None).items():
        ref.assert_within(n, x, want[n], bound[n])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,t,s,h,kv", [(70_001, 1, 1, 1, 1), (70_001, 1, 3, 2, 1), (300, 2, 2, 512, 256), (1, 3, 3, 4096, 4096)])
def test_many_sequences(b, t, s, h, kv, dtype):
    q, grad = (normal((b, t, h, 16), dtype, i) for i in range(2))
    k, v = (normal((b, s, kv, 16), dtype, i + 2) for i in range(2))
    got = run(q, k, v, grad, None)
    pick = torch.unique(torch.tensor([0, b // 3, b - 1]))
    heads = 16
    for at in (0, kv - min(kv, heads)):
        few = min(kv, heads)
        n = h // kv
        part = [q[pick][:, :, at * n:(at + few) * n], k[pick][:, :, at:at + few], v[pick][:, :, at:at + few],
                grad[pick][:, :, at * n:(at + few) * n]]
        want, bound = ref.attention(*part, None, 0.25, None)
        for name, x in got.items():
            x = x[pick][:, :, at * n:(at + few) * n] if name in ("out", "dq") else x[pick][:, :, at:at + few]
            ref.assert_within(name, x, want[name], bound[name])


@pytest.mark.parametrize("dtype,dim", [(torch.float32, d) for d in (4, 12, 20, 60, 68, 100, 124, 128)]
                         + [(t, d) for t in TYPES[1:] for d in (8, 24, 40, 56, 88, 104, 120)])
def test_head_widths(dim, dtype):
    """Grouped heads in a packed projection: neighbouring heads' channels follow at once."""
    t, h, kv = 150, 4, 2
    qkv = normal((2, t, (h + 2 * kv) * dim), dtype, dim)
    q, k, v = (x.reshape(2, t, -1, dim) for x in qkv.split([h * dim, kv * dim, kv * dim], -1))
    grad = normal((2, t, h, dim), dtype, 1)
    want, bound = ref.attention(q, k, v, grad, 70, dim ** -0.5, None)
    for n, x in run(q, k, v, grad, 70).items():
        ref.assert_within(n, x, want[n], bound[n])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("books,frames,entries,dim", [(3, 50, 20, 1), (2, 50, 20, 8191), (1, 9, 3, 65_536), (300, 5, 7, 8)])
def test_embedding_widths(books, frames, entries, dim, dtype):
    g = torch.Generator().manual_seed(dim)
    codes = torch.randint(-1, entries, (2, books, frames), generator=g)
    table, grad = normal((books, entries, dim), dtype, 1), normal((2, frames, dim), dtype, 2)
    want, bound = ref.embedding(codes, table, grad, 2.0)
    codes = codes.to(DEV)
    ref.assert_within("out", tr.code_embedding_forward(codes, table, 2.0), want["out"], bound["out"])
    ref.assert_within("dtable", tr.code_embedding_backward(grad, codes, table, 2.0), want["dtable"], bound["dtable"])
