"""What the training operators refuse, in Python and at the C ABI, without a GPU."""

from __future__ import annotations

import pytest
import torch

from fast_mimi_amd import _native as nat
from fast_mimi_amd import training as tr

X, W = torch.randn(4, 64), torch.ones(64)
Q = torch.randn(2, 5, 4, 64)
K = torch.randn(2, 5, 2, 64)
CODES, TABLE = torch.zeros(2, 3, 7, dtype=torch.int64), torch.randn(3, 16, 8)


@pytest.mark.parametrize("error,match,call", [
    (TypeError, "must be a tensor", lambda: tr.layer_norm([1.0])),
    (TypeError, "float32 or bfloat16 or float16", lambda: tr.layer_norm(X.double())),
    (ValueError, "last dimension", lambda: tr.layer_norm(torch.tensor(1.0))),
    (ValueError, "last dimension", lambda: tr.layer_norm(torch.empty(3, 0))),
    (ValueError, "weight must have shape", lambda: tr.layer_norm(X, W[:5])),
    (TypeError, "weight must be", lambda: tr.layer_norm(X, W.half())),
    (TypeError, "one type", lambda: tr.layer_norm(X.half(), W, W.half())),
    (ValueError, "eps", lambda: tr.layer_norm(X, W, W, -1.0)),
    (ValueError, "eps", lambda: tr.layer_norm(X, W, W, float("nan"))),
    (ValueError, "ROCm GPU", lambda: tr.layer_norm(X, W, W)),
    (ValueError, "grad must have x's shape", lambda: tr.layer_norm_backward(X[:2], X, X[:, 0], X[:, 0])),
    (TypeError, "grad must be", lambda: tr.layer_norm_backward(X.half(), X, X[:, 0], X[:, 0])),
    (ValueError, "layer_norm_forward returned", lambda: tr.layer_norm_backward(X, X, W, W)),
    (ValueError, r"\[batch, positions", lambda: tr.window_attention(Q[0], K, K)),
    (ValueError, "belong together", lambda: tr.window_attention(Q, K, K[:, :3])),
    (ValueError, "belong together", lambda: tr.window_attention(Q, K[..., :32], K[..., :32])),
    (ValueError, "last positions", lambda: tr.window_attention(Q, K[:, :3], K[:, :3])),
    (ValueError, "multiple of", lambda: tr.window_attention(Q[:, :, :3], K, K)),
    (ValueError, "head_dim", lambda: tr.window_attention(Q[..., :62], K[..., :62], K[..., :62])),
    (ValueError, "head_dim", lambda: tr.window_attention(Q[..., :4].half(), K[..., :4].half(), K[..., :4].half())),
    (ValueError, "head_dim", lambda: tr.window_attention(*[torch.randn(1, 2, 1, 132)] * 3)),
    (TypeError, "k must be", lambda: tr.window_attention(Q, K.half(), K.half())),
    (ValueError, "window", lambda: tr.window_attention(Q, K, K, 0)),
    (ValueError, "window", lambda: tr.window_attention(Q, K, K, True)),
    (ValueError, "window", lambda: tr.window_attention(Q, K, K, 2.5)),
    (ValueError, "scale", lambda: tr.window_attention(Q, K, K, scale=0.0)),
    (ValueError, "scale", lambda: tr.window_attention(Q, K, K, scale=float("inf"))),
    (ValueError, "scale", lambda: tr.window_attention(Q, K, K, scale=float("nan"))),
    (TypeError, "lengths must be", lambda: tr.window_attention(Q, K, K, lengths=torch.ones(2))),
    (TypeError, "lengths must be", lambda: tr.window_attention(Q, K, K, lengths=[5, 5])),
    (ValueError, "lengths must have", lambda: tr.window_attention(Q, K, K, lengths=torch.ones(3, dtype=torch.int32))),
    (ValueError, "ROCm GPU", lambda: tr.window_attention(Q, K, K)),
    (ValueError, "ROCm GPU", lambda: tr.window_attention(Q.requires_grad_(), K, K)),
    (ValueError, "grad must have q's shape", lambda: tr.window_attention_backward(Q[:1], Q, K, K, Q, Q[..., 0])),
    (ValueError, "window_attention_forward returned", lambda: tr.window_attention_backward(Q, Q, K, K, Q, Q[0, ..., 0])),
    (TypeError, "codes must be", lambda: tr.code_embedding(CODES.int(), TABLE)),
    (ValueError, "codes must be", lambda: tr.code_embedding(CODES[0], TABLE)),
    (ValueError, "table must be", lambda: tr.code_embedding(CODES, TABLE[0])),
    (ValueError, "table must be", lambda: tr.code_embedding(CODES, TABLE[:, :0])),
    (ValueError, "codebooks", lambda: tr.code_embedding(CODES, TABLE[:2])),
    (ValueError, "32768", lambda: tr.code_embedding(CODES[:, :1], torch.empty(1, 32769, 1))),
    (ValueError, "scale", lambda: tr.code_embedding(CODES, TABLE, float("nan"))),
    (ValueError, "ROCm GPU", lambda: tr.code_embedding(CODES, TABLE)),
    (ValueError, "grad must have shape", lambda: tr.code_embedding_backward(TABLE, CODES, TABLE)),
])
def test_python_refusals(error, match, call):
    with pytest.raises(error, match=match):
        call()


P = 0x10000  # never dereferenced


def attention(**change):
    a = dict(batch=1, queries=4, keys=4, heads=2, kv_heads=2, head_dim=64, window=4, scale=0.125, dtype=1, q=P, row=128, head=64,
             out=P)
    a.update(change)
    view = (a["q"], 1024, a["row"], a["head"])
    return nat.library().fm_attention_forward(
        *view, P, 1024, 128, 64, P, 1024, 128, 64, None, a["batch"], a["queries"], a["keys"], a["heads"], a["kv_heads"],
        a["head_dim"], a["window"], a["scale"], a["dtype"], a["out"], P, None, 0, None)


@pytest.mark.skipif(not nat.LIBRARY_PATH.is_file(), reason="library not built")
@pytest.mark.parametrize("status,change", [
    (1000, dict(batch=-1)), (1000, dict(queries=5)), (1000, dict(heads=3)), (1000, dict(kv_heads=0)), (1000, dict(window=0)),
    (1000, dict(scale=0.0)), (1000, dict(scale=float("nan"))), (1000, dict(dtype=3)), (1000, dict(q=None)), (1000, dict(out=None)),
    (1002, dict(head_dim=136)), (1002, dict(head_dim=60)), (1002, dict(q=P + 2)), (1002, dict(row=129)), (1002, dict(row=1 << 40)),
    (1002, dict(head=-64)), (1002, dict(out=P + 4)), (1002, dict(queries=1 << 30, keys=1 << 30)),
    (1000, dict(scale=3e38)), (1002, dict(keys=2_097_121)), (1002, dict(batch=1 << 23)), (1002, dict(heads=1 << 21, kv_heads=1)),
    (1001, dict(queries=1, keys=100_000, window=100_000)),
    (0, dict(batch=0)), (0, dict(queries=0)),
])
def test_attention_abi_refusals(status, change):
    assert attention(**change) == status


@pytest.mark.skipif(not nat.LIBRARY_PATH.is_file(), reason="library not built")
def test_other_abi_refusals():
    lib = nat.library()
    forward, backward = lib.fm_layer_norm_forward, lib.fm_layer_norm_backward
    assert forward(None, 64, None, None, 4, 64, 1e-5, 0, 0, P, P, P, None) == 1000
    assert forward(P, 64, None, None, 4, 0, 1e-5, 0, 0, P, P, P, None) == 1000
    assert forward(P, 64, None, None, 4, 64, 1e-5, 0, 1, P, P, P, None) == 1000
    assert forward(P, 64, None, None, 1 << 40, 64, 1e-5, 0, 0, P, P, P, None) == 1002
    assert forward(None, 64, None, None, 0, 64, 1e-5, 0, 0, None, None, None, None) == 0
    assert backward(P, 64, P, 64, P, P, P, 400, 64, 0, 0, P, P, P, None, 0, None) == 1001
    assert backward(P, 64, P, 64, P, P, P, 400, 64, 0, 0, P, P, P, None, 1 << 20, None) == 1000
    assert backward(P, 64, None, 64, P, P, P, 4, 64, 0, 0, P, P, P, P, 1 << 20, None) == 1000
    embed, gradient = lib.fm_code_embedding, lib.fm_code_embedding_backward
    assert embed(P, 8, 8, 1, 1, 8, None, 16, 8, 1.0, 0, P, None) == 1000
    assert embed(P, 8, 8, 1, 1, 8, P, 40_000, 8, 1.0, 0, P, None) == 1002
    assert embed(P, 8, 8, 1, 0, 8, P, 16, 8, 1.0, 0, P, None) == 1000
    assert embed(P, -8, 8, 1, 1, 8, P, 16, 8, 1.0, 0, P, None) == 1000
    assert gradient(P, 8, P, 8, 8, 1, 1, 8, 16, 8, 1.0, 0, P, None, 0, None) == 1001
    assert gradient(P, 8, P, 8, 8, 1, 1, 8, 16, 8, 1.0, 0, None, P, 1 << 20, None) == 1000
    assert gradient(P, 8, P, 8, 8, 1 << 20, 1, 1 << 20, 16, 8, 1.0, 0, P, P, 1 << 20, None) == 1002


@pytest.mark.skipif(not nat.LIBRARY_PATH.is_file(), reason="library not built")
def test_workspace_queries_are_host_only():
    lib = nat.library()
    assert lib.fm_attention_forward_workspace_bytes(16, 250, 250, 8, 8, 64, 250) == 0
    assert lib.fm_attention_forward_workspace_bytes(1, 1, 8000, 8, 8, 64, 8000) > 0
    assert lib.fm_attention_forward_workspace_bytes(1, 9, 8, 8, 8, 64, 8) == 0
    assert 0 < lib.fm_layer_norm_backward_workspace_bytes(100, 512) <= 100 * 4096
    assert lib.fm_layer_norm_backward_workspace_bytes(0, 512) == 0
    assert lib.fm_code_embedding_backward_workspace_bytes(1, 8, 13, 2048, 256) > 8 * 2049 * 4
