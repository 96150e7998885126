"""Forward-mode derivatives: the training operators have none, and say so instead
of returning outputs without a tangent."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fw

from fast_mimi_amd import training as tr

X, W = torch.randn(4, 64), torch.ones(64)
Q = torch.randn(2, 5, 2, 64)
CODES, TABLE = torch.zeros(2, 3, 7, dtype=torch.int64), torch.randn(3, 16, 8)

CALLS = [
    (X, lambda x: tr.layer_norm(x, W, W)),
    (W, lambda w: tr.layer_norm(X, w)),
    (W, lambda b: tr.layer_norm(X, None, b)),
    (Q, lambda q: tr.window_attention(q, Q, Q)),
    (Q, lambda k: tr.window_attention(Q, k, Q)),
    (Q, lambda v: tr.window_attention(Q, Q, v, 3)),
    (TABLE, lambda t: tr.code_embedding(CODES, t)),
    (X, lambda g: tr.layer_norm_backward(g, X, X[:, 0].contiguous(), X[:, 0].contiguous(), W)),
    (Q, lambda g: tr.window_attention_backward(g, Q, Q, Q, Q, Q[..., 0].contiguous())),
    (torch.randn(2, 7, 8), lambda g: tr.code_embedding_backward(g, CODES, TABLE)),
]


@pytest.mark.parametrize("at,call", CALLS)
def test_dual_tensors_are_refused(at, call):
    with fw.dual_level():
        for requires in (False, True):
            x = at.clone().requires_grad_(requires)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(fw.make_dual(x, torch.ones_like(at)))


@pytest.mark.parametrize("at,call", CALLS)
def test_jvp_is_refused(at, call):
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(call, (at,), (torch.ones_like(at),))


@pytest.mark.parametrize("at,call", CALLS)
def test_a_level_alone_refuses_nothing(at, call):
    """Tensors without a tangent go on to the next check."""
    with fw.dual_level(), pytest.raises(ValueError, match="ROCm GPU"):
        call(at)
