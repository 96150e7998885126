"""Sizes that the C ABI's 32 bits cannot hold are refused before anything is launched, without a GPU: they would
arrive there as other, small ones.  The tensors are views of single elements."""

from __future__ import annotations

import pytest
import torch

from fast_mimi_amd import _native as nat
from fast_mimi_amd import quantized as qz
from fast_mimi_amd import training as tr

FAR = (1 << 32) + 64  # its low 32 bits are 64


def wide(*shape, dtype=torch.float32):
    return torch.zeros(1).to(dtype).reshape((1,) * len(shape)).expand(shape)


def scales(*shape):
    return torch.full((1,) * len(shape), 127, dtype=torch.uint8).view(torch.float8_e8m0fnu).expand(shape)


F8 = torch.float8_e4m3fn
ONE = torch.ones(1)


@pytest.mark.parametrize("call", [
    lambda: tr.rms_norm(wide(1, FAR)),
    lambda: tr.rms_norm_backward(wide(1, FAR), wide(1, FAR), ONE),
    lambda: tr.layer_norm(wide(1, FAR)),
    lambda: tr.layer_norm_backward(wide(1, FAR), wide(1, FAR), ONE, ONE),
    lambda: tr.rotary(wide(1, 1, FAR, 4), None, torch.ones(2, dtype=torch.float64)),
    lambda: tr.rotary(wide(1, 1, 1, 4), wide(1, 1, FAR, 4), torch.ones(2, dtype=torch.float64)),
    lambda: tr.cross_attention(wide(1, 1, 1, 64), wide(1, FAR, 1, 64), wide(1, FAR, 1, 64)),
    lambda: tr.cross_attention(wide(1, FAR, 1, 64), wide(1, 2, 1, 64), wide(1, 2, 1, 64)),
    lambda: tr.cross_attention(wide(FAR, 1, 1, 64), wide(FAR, 2, 1, 64), wide(FAR, 2, 1, 64)),
    lambda: tr.cross_attention(wide(1, 1, FAR, 64), wide(1, 2, 1, 64), wide(1, 2, 1, 64)),
    lambda: tr.cross_attention_backward(wide(1, 1, 1, 64), wide(1, 1, 1, 64), wide(1, FAR, 1, 64), wide(1, FAR, 1, 64),
                                        wide(1, 1, 1, 64), wide(1, 1, 1)),
    lambda: tr.window_attention(wide(1, 1, 1, 64), wide(1, FAR, 1, 64), wide(1, FAR, 1, 64), 8),
    lambda: tr.code_embedding(wide(FAR, 1, 1, dtype=torch.int64), torch.ones(1, 4, 8)),
    lambda: tr.code_embedding(wide(1, 1, FAR, dtype=torch.int64), torch.ones(1, 4, 8)),
    lambda: tr.code_embedding(wide(1, 1, 1, dtype=torch.int64), wide(1, 4, FAR)),
    lambda: qz.quantize(wide(1, FAR)),
    lambda: qz.quantize_weight(wide(FAR, 16)),
    lambda: qz.quantize_weight(wide(1, FAR)),
    lambda: qz.rms_norm(wide(1, FAR)),
    lambda: qz.linear(wide(1, FAR, dtype=F8), scales(1, -(-FAR // 128)), wide(1, FAR, dtype=F8), scales(1, -(-FAR // 128))),
    lambda: qz.linear(wide(1, 16, dtype=F8), scales(1, 1), wide(FAR, 16, dtype=F8), scales(-(-FAR // 128), 1)),
])
def test_sizes_beyond_32_bits(call):
    with pytest.raises(ValueError, match="below 2\\^31"):
        call()


@pytest.mark.skipif(not nat.LIBRARY_PATH.is_file(), reason="library not built")
def test_why():
    """The binding passes the low 32 bits on."""
    query = nat.library().fm_cross_attention_forward_workspace_bytes
    assert query(1, 1, (1 << 32) + 5000, 1, 1, 64) == query(1, 1, 5000, 1, 1, 64) > 0
