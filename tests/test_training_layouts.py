"""Strides of single items say nothing: views that have odd ones are taken."""

from __future__ import annotations

import pytest
import torch

from fast_mimi_amd import training as tr

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def odd_views(dtype, device="cpu"):
    """[B, N, H, D] views at an address that is no multiple of 16 bytes, with
    strides that are no multiple of one either where a dimension has one item."""
    room = torch.arange(40_000, device=device).remainder(97).to(dtype)
    return [
        room.as_strided((1, 50, 1, 64), (3201, 64, 64, 1), 1),
        room.as_strided((1, 50, 1, 64), (3201, 64, 7, 1), 1),
        room.as_strided((1, 50, 2, 64), (12345, 128, 64, 1), 1),
        room.as_strided((3, 1, 2, 64), (128, 129, 64, 1), 1),
        room.as_strided((1, 1, 1, 64), (1, 3, 5, 1), 1),
        room.as_strided((1, 1, 2, 64), (1, 3, 64, 1), 3),
        room.as_strided((1, 50, 1, 64), (3, 65, 5, 1), 0),
        room.as_strided((2, 50, 1, 64), (3201, 64, 64, 1), 0),
        room.as_strided((1, 50, 1, 64), (3201, 64, 3, 1), 0),  # aligned: read in place
    ]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("i", range(9))
def test_heads_are_aligned(i, dtype):
    view = odd_views(dtype)[i]
    t, *strides = tr._heads(view)
    unit = 16 // t.element_size()
    assert torch.equal(t, view)
    assert t.data_ptr() % 16 == 0 and t.stride(3) == 1 and all(s % unit == 0 and s >= 0 for s in strides)
    for size, own, given in zip(t.shape, t.stride(), strides):
        assert size == 1 or own == given


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("i", range(9))
def test_attention_of_odd_views(i, dtype):
    x = odd_views(dtype, "cuda")[i]
    x.div_(97)
    plain = torch.empty(x.shape, dtype=dtype, device="cuda").copy_(x)
    want, lse = tr.window_attention_forward(plain, plain, plain, 20)
    out, _ = tr.window_attention_forward(x, x, x, 20)
    assert torch.equal(out, want)
    got = tr.window_attention_backward(x, x, x, x, out, lse, 20)
    for a, b in zip(got, tr.window_attention_backward(plain, plain, plain, plain, want, lse, 20)):
        assert torch.equal(a, b)


def test_pitches_at_the_abi():
    """A row or head pitch beyond what a tile's 32-bit offsets reach is refused; the
    largest ones are not (an empty batch, so that nothing runs)."""
    from fast_mimi_amd import _native as nat

    if not nat.LIBRARY_PATH.is_file():
        pytest.skip("library not built")
    p = 0x10000  # never dereferenced

    def status(row, head, heads=4, dtype=1):
        view, keys = (p, 0, row, head), (p, 0, 64, 64)
        return nat.library().fm_attention_forward(*view, *keys, *keys, None, 0, 4, 4, heads, 1, 64, 4, 0.125, dtype, p, p, None, 0,
                                                  None)

    row, head = (2 ** 31 - 1) // 2 // 256, (2 ** 31 - 1) // 2 // 2 // 4
    assert status(row // 8 * 8, head // 8 * 8) == 0
    assert status(row // 8 * 8 + 8, 64) == 1002 and status(64, head // 8 * 8 + 8) == 1002
    assert status(row // 2 // 4 * 4, head // 2 // 4 * 4, dtype=0) == 0
    assert status(row // 2 // 4 * 4 + 4, 64, dtype=0) == 1002
