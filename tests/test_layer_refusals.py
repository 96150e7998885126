"""What RMS norm, rotary positions, cross attention and the 8-bit operators refuse, in Python
and at the C ABI, without a GPU."""

from __future__ import annotations

import pytest
import torch

from fast_mimi_amd import _native as nat
from fast_mimi_amd import quantized as qz
from fast_mimi_amd import training as tr

X, W, R = torch.randn(4, 64), torch.ones(64), torch.ones(4)
Q, K = torch.randn(2, 5, 4, 64), torch.randn(2, 7, 2, 64)
F = tr.rotary_frequencies(64)
LSE = torch.zeros(2, 5, 4)
N = torch.ones(2, dtype=torch.int32)
X8, W8 = torch.zeros(4, 256).to(torch.float8_e4m3fn), torch.zeros(100, 256).to(torch.float8_e4m3fn)


def scales(*shape):
    return torch.full(shape, 127, dtype=torch.uint8).view(torch.float8_e8m0fnu)


XS, WS = scales(4, 2), scales(1, 2)


@pytest.mark.parametrize("error,match,call", [
    (TypeError, "must be a tensor", lambda: tr.rms_norm([1.0])),
    (TypeError, "float32 or bfloat16 or float16", lambda: tr.rms_norm(X.double())),
    (ValueError, "last dimension", lambda: tr.rms_norm(torch.tensor(1.0))),
    (ValueError, "last dimension", lambda: tr.rms_norm(torch.empty(3, 0))),
    (ValueError, "weight must have shape", lambda: tr.rms_norm(X, W[:5])),
    (TypeError, "weight must be float32", lambda: tr.rms_norm(X, W.half())),
    (ValueError, "residual must have", lambda: tr.rms_norm(X, W, X[:2])),
    (TypeError, "residual must be float32", lambda: tr.rms_norm(X, W, X.half())),
    (TypeError, "residual must be", lambda: tr.rms_norm(X.half(), W, X.bfloat16())),
    (ValueError, "eps", lambda: tr.rms_norm(X, W, None, -1.0)),
    (ValueError, "eps", lambda: tr.rms_norm(X, W, None, float("nan"))),
    (ValueError, "ROCm GPU", lambda: tr.rms_norm(X, W, X)),
    (ValueError, "ROCm GPU", lambda: tr.rms_norm(X.requires_grad_(), W)),
    (ValueError, "grad must have x's shape", lambda: tr.rms_norm_backward(X[:2], X, R)),
    (TypeError, "x must be", lambda: tr.rms_norm_backward(X, X.half(), R)),
    (TypeError, "x must be", lambda: tr.rms_norm_backward(X.half(), X, R, None, X)),
    (ValueError, "residual must have", lambda: tr.rms_norm_backward(X, X, R, None, X[:1])),
    (ValueError, "rms_norm_forward returned", lambda: tr.rms_norm_backward(X, X, W)),
    (TypeError, "rstd must be", lambda: tr.rms_norm_backward(X, X, R.double())),
    (TypeError, "grad_h must be", lambda: tr.rms_norm_backward(X, X, R, None, None, X.half())),
    (ValueError, "grad_h must have", lambda: tr.rms_norm_backward(X, X, R, None, None, X[:1])),
    (ValueError, r"\[batch, positions", lambda: tr.rotary(Q[0], None, F)),
    (ValueError, "belong together", lambda: tr.rotary(Q, K, F)),
    (ValueError, "belong together", lambda: tr.rotary(Q, Q[..., :32], F[:8])),
    (TypeError, "k must be", lambda: tr.rotary(Q, Q.half(), F)),
    (TypeError, "frequencies must be float64", lambda: tr.rotary(Q, None, F.float())),
    (ValueError, r"frequencies must be \[pairs\]", lambda: tr.rotary(Q, None, F[None])),
    (ValueError, r"frequencies must be \[pairs\]", lambda: tr.rotary(Q, None, F[:0])),
    (ValueError, r"frequencies must be \[pairs\]", lambda: tr.rotary(Q[..., :62], None, F)),
    (TypeError, "positions must be", lambda: tr.rotary(Q, None, F, torch.arange(5.0))),
    (TypeError, "positions must be a tensor", lambda: tr.rotary(Q, None, F, True)),
    (TypeError, "positions must be a tensor", lambda: tr.rotary(Q, None, F, 2.5)),
    (ValueError, "positions must have", lambda: tr.rotary(Q, None, F, torch.arange(4))),
    (ValueError, "53 bits", lambda: tr.rotary(Q, None, F, (1 << 53) - 4)),
    (ValueError, "53 bits", lambda: tr.rotary(Q, None, F, -(1 << 53) - 1)),
    (ValueError, "head_dim", lambda: tr.rotary(torch.empty(1, 1, 1, 514), None, F)),
    (ValueError, "scale", lambda: tr.rotary(Q, None, F, scale=float("inf"))),
    (ValueError, "positions in all", lambda: tr.rotary(torch.empty(1, 1, 1, 1).expand(4097, 4096, 1, 2), None, F[:1])),
    (ValueError, "ROCm GPU", lambda: tr.rotary(Q, Q, F)),
    (ValueError, "dim must be", lambda: tr.rotary_frequencies(7)),
    (ValueError, "dim must be", lambda: tr.rotary_frequencies(0)),
    (ValueError, "base and factor", lambda: tr.rotary_frequencies(8, base=-1.0)),
    (ValueError, "base and factor", lambda: tr.rotary_frequencies(8, factor=float("nan"))),
    (ValueError, "method must be", lambda: tr.rotary_frequencies(8, method="other")),
    (ValueError, "slower", lambda: tr.rotary_frequencies(2, factor=2.0, method="base")),
    (ValueError, "context", lambda: tr.rotary_frequencies(8, factor=2.0, method="ramp")),
    (ValueError, "fast > slow", lambda: tr.rotary_frequencies(8, factor=2.0, method="ramp", context=100, fast=1.0, slow=1.0)),
    (ValueError, r"\[batch, positions", lambda: tr.cross_attention(Q[0], K, K)),
    (ValueError, "belong together", lambda: tr.cross_attention(Q, K, K[:, :3])),
    (ValueError, "belong together", lambda: tr.cross_attention(Q[:1], K, K)),
    (ValueError, "multiple of", lambda: tr.cross_attention(Q[:, :, :3], K, K)),
    (ValueError, "head_dim", lambda: tr.cross_attention(Q[..., :62], K[..., :62], K[..., :62])),
    (TypeError, "k must be", lambda: tr.cross_attention(Q, K.half(), K.half())),
    (ValueError, "scale", lambda: tr.cross_attention(Q, K, K, 0.0)),
    (TypeError, "key_lengths must be", lambda: tr.cross_attention(Q, K, K, key_lengths=N.long())),
    (ValueError, "key_lengths must have", lambda: tr.cross_attention(Q, K, K, key_lengths=N[:1])),
    (TypeError, "query_lengths must be", lambda: tr.cross_attention(Q, K, K, query_lengths=[1, 2])),
    (ValueError, "query_lengths must have", lambda: tr.cross_attention(Q, K, K, query_lengths=N[None])),
    (ValueError, "ROCm GPU", lambda: tr.cross_attention(Q, K, K, key_lengths=N)),
    (ValueError, "grad must have q's shape", lambda: tr.cross_attention_backward(Q[:1], Q, K, K, Q, LSE)),
    (ValueError, "cross_attention_forward returned", lambda: tr.cross_attention_backward(Q, Q, K, K, Q, LSE[0])),
    (TypeError, "must be a tensor", lambda: qz.quantize(3.0)),
    (TypeError, "float32 or bfloat16 or float16", lambda: qz.quantize(X8)),
    (ValueError, "last dimension", lambda: qz.quantize(torch.empty(3, 0))),
    (ValueError, "ROCm GPU", lambda: qz.quantize(X.detach())),
    (ValueError, r"weight must be \[out, in\]", lambda: qz.quantize_weight(W)),
    (ValueError, r"weight must be \[out, in\]", lambda: qz.quantize_weight(torch.empty(0, 4))),
    (ValueError, "residual must have", lambda: qz.rms_norm(X.detach(), None, X.detach()[:2])),
    (ValueError, "ROCm GPU", lambda: qz.rms_norm(X.detach())),
    (RuntimeError, "no gradient", lambda: qz.quantize(torch.ones(3, requires_grad=True))),
    (RuntimeError, "no gradient", lambda: qz.rms_norm(X.detach(), torch.ones(64, requires_grad=True))),
    (TypeError, "x must be float8_e4m3fn", lambda: qz.linear(X, XS, W8, WS)),
    (TypeError, "x_scale must be float8_e8m0fnu", lambda: qz.linear(X8, XS.float(), W8, WS)),
    (TypeError, "weight must be float8_e4m3fn", lambda: qz.linear(X8, XS, W8.float(), WS)),
    (TypeError, "dtype must be", lambda: qz.linear(X8, XS, W8, WS, torch.float64)),
    (ValueError, r"weight must be \[out, in\]", lambda: qz.linear(X8, XS, W8[0], WS)),
    (ValueError, r"x must be \[\.\.\., 256\]", lambda: qz.linear(X8[:, :128], XS, W8, WS)),
    (ValueError, "multiple of 16", lambda: qz.linear(X8[:, :250], XS, W8[:, :250], WS)),
    (ValueError, "x_scale must have", lambda: qz.linear(X8, XS[:, :1], W8, WS)),
    (ValueError, "weight_scale must have", lambda: qz.linear(X8, XS, W8, XS)),
    (ValueError, "ROCm GPU", lambda: qz.linear(X8, XS, W8, WS)),
    (RuntimeError, "no gradient", lambda: qz.linear(X8, XS, W8.detach().requires_grad_(), WS)),
    (ValueError, "no gradient", lambda: tr.rotary(Q, Q, F.clone().requires_grad_())),
])
def test_python_refusals(error, match, call):
    with pytest.raises(error, match=match):
        call()


def test_forward_mode_is_refused():
    with torch.autograd.forward_ad.dual_level():
        x = torch.autograd.forward_ad.make_dual(X.detach(), X.detach())
        q = torch.autograd.forward_ad.make_dual(Q, Q)
        for call in (lambda: tr.rms_norm(x), lambda: tr.rotary(q, None, F), lambda: tr.cross_attention(q, K, K), lambda: qz.quantize(x)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_frequencies():
    """Each method against its formula; the stretched ends are where they belong."""
    i = torch.arange(32, dtype=torch.float64)
    plain = 10_000.0 ** (-2 * i / 64)
    assert torch.allclose(F, plain, rtol=1e-15)
    assert torch.allclose(tr.rotary_frequencies(64, factor=4.0), plain / 4, rtol=1e-15)
    base = tr.rotary_frequencies(64, factor=4.0, method="base")
    assert base[0] == 1 and abs(base[-1] / (plain[-1] / 4) - 1) < 1e-12 and (base <= plain).all()
    ramp = tr.rotary_frequencies(64, factor=4.0, method="ramp", context=2000)
    turns = 2000 * plain / (2 * torch.pi)
    assert torch.equal(ramp[turns > 32], plain[turns > 32]) and torch.allclose(ramp[turns < 1], plain[turns < 1] / 4, rtol=1e-15)
    between = (turns < 32) & (turns > 1)
    assert between.any() and (ramp[between] < plain[between]).all() and (ramp[between] > plain[between] / 4).all()
    # Without a factor as they were, but for the roundings of the two parts' sum and its product.
    assert torch.allclose(tr.rotary_frequencies(64, method="ramp", context=10), F, rtol=2 ** -51, atol=0)


P = 0x10000  # never dereferenced
built = pytest.mark.skipif(not nat.LIBRARY_PATH.is_file(), reason="library not built")


@built
def test_norm_abi_refusals():
    lib = nat.library()

    def forward(x=P, residual=P, rows=4, channels=64, eps=1e-5, dtype=1, stream=0, weight=0, y=P, h=P, rstd=P):
        return lib.fm_rms_norm_forward(x, 64, residual, 64, P, rows, channels, eps, dtype, stream, weight, y, h, rstd, None)

    for change in (dict(x=None), dict(y=None), dict(h=None), dict(rstd=None), dict(rows=-1), dict(channels=0), dict(eps=-1.0),
                   dict(eps=float("nan")), dict(dtype=3), dict(dtype=-1), dict(stream=2), dict(weight=2)):
        assert forward(**change) == 1000, change
    assert forward(rows=(1 << 31) - 1) == 1002 and forward(channels=(1 << 26) + 1) == 1002
    assert forward(rows=0, x=None) == 0

    def backward(dy=P, x=P, residual=P, rows=400, channels=64, dgamma=P, dres=P, ws=P, size=1 << 20):
        return lib.fm_rms_norm_backward(dy, 64, x, 64, residual, 64, P, P, None, 0, rows, channels, 1, 1, 1, None, dres, dgamma, ws,
                                        size, None)

    assert backward(x=None, residual=None) == 1000 and backward(dy=None) == 1000 and backward(dres=None) == 1000
    assert backward(ws=None) == 1000 and backward(ws=None, size=0) == 1001 and backward(size=100) == 1001
    assert backward(rows=0, dgamma=None) == 0
    assert lib.fm_rms_norm_quantized(P, 64, None, 0, P, 4, 64, 1e-5, 1, 1, 1, P, None, None, None) == 1000
    assert lib.fm_rms_norm_quantized(P, 64, P, 64, P, 4, 64, 1e-5, 1, 1, 1, P, P, None, None) == 1000
    assert lib.fm_quantize_rows(P, 64, 4, 64, 5, P, P, None) == 1000 and lib.fm_quantize_rows(None, 64, 4, 64, 0, P, P, None) == 1000
    assert lib.fm_quantize_rows(None, 64, 0, 64, 0, None, None, None) == 0
    assert lib.fm_quantize_weight(P, 0, 64, 0, P, P, None) == 1000 and lib.fm_quantize_weight(P, 64, 64, 0, None, P, None) == 1000
    assert lib.fm_quantize_weight(P, 128 * 65536, 64, 0, P, P, None) == 1002


@built
def test_rotary_abi_refusals():
    lib = nat.library()

    def call(q=P, heads=4, k=P, kv=2, freq=P, pos=P, size=8, batch=2, length=3, dim=64, rotated=64, scale=1.0, dtype=1, q_out=P, k_out=P):
        return lib.fm_rotary(q, 64, 64, 64, heads, k, 64, 64, 64, kv, freq, pos, 3, size, 0, batch, length, dim, rotated, 0, scale, 0,
                             dtype, q_out, k_out, None)

    for change in (dict(q=None), dict(k=None), dict(freq=None), dict(q_out=None), dict(k_out=None), dict(size=2), dict(batch=-1),
                   dict(length=-1), dict(heads=-1), dict(dim=0), dict(rotated=66), dict(rotated=63), dict(rotated=-2), dict(dtype=3),
                   dict(scale=float("nan"))):
        assert call(**change) == 1000, change
    assert call(dim=514) == 1002 and call(batch=1 << 13, length=1 << 12) == 1002 and call(heads=65535) == 1002
    assert call(batch=0, q=None) == 0 and call(length=0) == 0 and call(heads=0, kv=0, q=None, k=None) == 0


@built
def test_cross_attention_abi_refusals():
    lib = nat.library()

    def forward(q=P, k=P, batch=1, queries=4, keys=6, heads=2, kv=2, dim=64, scale=0.125, dtype=1, out=P, lse=P, row=128, ws=None,
                size=0):
        return lib.fm_cross_attention_forward(q, 1024, row, 64, k, 1024, 128, 64, P, 1024, 128, 64, None, None, batch, queries, keys,
                                              heads, kv, dim, scale, dtype, out, lse, ws, size, None)

    for change in (dict(q=None), dict(k=None), dict(out=None), dict(lse=None), dict(batch=-1), dict(queries=-1), dict(keys=-1),
                   dict(heads=3), dict(kv=0), dict(scale=0.0), dict(scale=float("nan")), dict(scale=3e38), dict(dtype=3)):
        assert forward(**change) == 1000, change
    for change in (dict(dim=136), dict(dim=60), dict(q=P + 2), dict(row=129), dict(row=1 << 40), dict(out=P + 4), dict(keys=2_097_121),
                   dict(queries=1 << 30), dict(batch=1 << 23)):
        assert forward(**change) == 1002, change
    assert forward(queries=1, keys=100_000) == 1001 and forward(queries=1, keys=100_000, ws=P + 4, size=1 << 30) == 1002
    assert forward(batch=0, q=None) == 0 and forward(queries=0, q=None) == 0

    def backward(dout=P, k=P, queries=4, keys=6, stats=P, dk=P, ws=None, size=0):
        return lib.fm_cross_attention_backward(dout, 1024, 128, 64, P, 1024, 128, 64, k, 1024, 128, 64, P, 1024, 128, 64, P, P, None,
                                               None, 1, queries, keys, 2, 2, 64, 0.125, 1, P, dk, P, stats, ws, size, None)

    assert backward(dout=None) == 1000 and backward(stats=None) == 1000 and backward(dk=None) == 1000 and backward(dk=P + 4) == 1002
    assert backward(queries=4000) == 1001 and backward(keys=4000) == 1001
    assert backward(queries=0) == 1000 and backward(queries=0, keys=0) == 0


@built
def test_linear_abi_refusals():
    lib = nat.library()

    def call(x=P, w=P, rows=64, k=256, n=100, dtype=1, y=P, ws=None, size=0):
        return lib.fm_linear_fp8(x, P, w, P, rows, k, n, dtype, y, ws, size, None)

    for change in (dict(x=None), dict(w=None), dict(y=None), dict(rows=-1), dict(k=0), dict(n=0), dict(dtype=3)):
        assert call(**change) == 1000, change
    for change in (dict(k=250), dict(k=1 << 23), dict(x=P + 8), dict(w=P + 1), dict(y=P + 4), dict(rows=(1 << 24) + 1),
                   dict(n=(1 << 24) + 1), dict(rows=1 << 24, n=1 << 20)):
        assert call(**change) == 1002, change
    need = lib.fm_linear_fp8_workspace_bytes(64, 8192, 100)
    assert need > 0 and call(k=8192) == 1001 and call(k=8192, ws=P, size=need - 1) == 1001 and call(k=8192, ws=P + 4, size=need) == 1002
    assert call(rows=0, x=None) == 0


@built
def test_workspace_queries_are_host_only():
    lib = nat.library()
    assert lib.fm_rms_norm_backward_workspace_bytes(13, 512) == 0 and lib.fm_rms_norm_backward_workspace_bytes(0, 64) == 0
    assert 0 < lib.fm_rms_norm_backward_workspace_bytes(100, 512) <= 100 * 2048
    assert lib.fm_linear_fp8_workspace_bytes(8192, 8192, 8192) == 0 and lib.fm_linear_fp8_workspace_bytes(0, 64, 64) == 0
    assert lib.fm_cross_attention_forward_workspace_bytes(1, 1, 8000, 8, 8, 64) > 0
    assert lib.fm_cross_attention_backward_workspace_bytes(1, 4000, 64, 8, 8, 64) > 0
    assert lib.fm_cross_attention_backward_workspace_bytes(16, 2500, 2500, 8, 8, 64) == 0
    assert lib.fm_cross_attention_backward_workspace_bytes(1, 9, 8, 8, 3, 64) == 0
