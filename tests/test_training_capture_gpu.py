"""The differentiable training functions in hipGraphs: after a warm-up on a side
stream whose autograd graph stays alive, and through torch's own helper."""

from __future__ import annotations

import pytest
import torch

from fast_mimi_amd import training as tr

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Layer(torch.nn.Module):
    def __init__(self):
        super().__init__()
        g = torch.Generator().manual_seed(1)
        self.weight = torch.nn.Parameter((1 + 0.1 * torch.randn(128, generator=g)).to(DEV))
        self.bias = torch.nn.Parameter((0.1 * torch.randn(128, generator=g)).to(DEV))

    def forward(self, x):
        b, t, c = x.shape
        y = tr.layer_norm(x, self.weight, self.bias)
        heads = y.view(b, t, 2, 64)
        return x + tr.window_attention(heads, heads, heads, 20).reshape(b, t, c)


def by_hand(layer, x, grad):
    """Output and gradients from the functions without autograd."""
    b, t, c = x.shape
    w, bias = layer.weight.detach(), layer.bias.detach()
    y, mean, rstd = tr.layer_norm_forward(x, w, bias)
    heads = y.view(b, t, 2, 64)
    out, lse = tr.window_attention_forward(heads, heads, heads, 20)
    dq, dk, dv = tr.window_attention_backward(grad.view(b, t, 2, 64), heads, heads, heads, out, lse, 20)
    dx, dw, db = tr.layer_norm_backward((dq + dk + dv).view(b, t, c), x, mean, rstd, w, bias)
    return x + out.view(b, t, c), grad + dx, dw, db


def inputs(seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(2, 50, 128, generator=g, device=DEV) for _ in range(2)]


def close(got, want):
    # Sums of the same terms in other orders, in FP32.
    for a, b in zip(got, want):
        assert (a - b).abs().max() <= 1e-5 * b.abs().max()


def test_a_side_stream_warm_up_may_stay_alive():
    layer = Layer()
    x, grad = inputs(1)
    x.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            alive = layer(x)  # the last one's graph stays
            alive.backward(grad)
    torch.cuda.current_stream().wait_stream(side)
    x.grad = None
    layer.zero_grad(set_to_none=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = layer(x)
        out.backward(grad)
    for seed in (2, 3, 4):
        with torch.no_grad():
            for to, fresh in zip((x, grad), inputs(seed)):
                to.copy_(fresh)
        g.replay()
        torch.cuda.synchronize()
        close((out, x.grad, layer.weight.grad, layer.bias.grad), by_hand(layer, x.detach(), grad))
    assert alive.grad_fn is not None


def test_make_graphed_callables():
    layer = Layer()
    x, grad = inputs(1)
    graphed = torch.cuda.make_graphed_callables(layer, (x.requires_grad_(),))
    for seed in (2, 3, 4):
        x, grad = inputs(seed)
        leaf = x.clone().requires_grad_()
        layer.zero_grad(set_to_none=True)
        out = graphed(leaf)
        out.backward(grad)
        torch.cuda.synchronize()
        close((out, leaf.grad, layer.weight.grad, layer.bias.grad), by_hand(layer, x, grad))


def test_a_held_accumulator_of_the_default_stream_is_refused():
    """The graph is gone, the accumulator and its stream are not."""
    w = torch.ones(64, device=DEV, requires_grad=True)
    x = torch.randn(8, 64, device=DEV)
    holder = w.view_as(w).grad_fn.next_functions[0][0]
    y = tr.layer_norm(x, w)
    del y
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="default stream"):
        with torch.cuda.graph(g):
            tr.layer_norm(x, w)
    del holder
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = tr.layer_norm(x, w)
        (dw,) = torch.autograd.grad(y, w, x)
    g.replay()
    torch.cuda.synchronize()
    _, mean, rstd = tr.layer_norm_forward(x, w.detach())
    assert torch.equal(dw, tr.layer_norm_backward(x, x, mean, rstd, w.detach())[1])


def test_a_leaf_first_used_in_a_capture_may_be_captured_again():
    """Also after an eager call on the default stream: the accumulator is the capture's."""
    w = torch.ones(64, device=DEV, requires_grad=True)
    x = torch.randn(8, 64, device=DEV)
    tr.layer_norm(x, w.detach())
    torch.cuda.synchronize()
    graphs, kept = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = tr.layer_norm(x, w)
            kept.append((y, *torch.autograd.grad(y, w, x)))
        graphs.append(g)
        kept.append((tr.layer_norm(x, w),))
    for seed in (1, 2, 3):
        x.copy_(torch.randn(8, 64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)))
        want, mean, rstd = tr.layer_norm_forward(x, w.detach())
        dw = tr.layer_norm_backward(x, x, mean, rstd, w.detach())[1]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for y, got in (kept[0], kept[2]):
            assert torch.equal(y, want) and torch.equal(got, dw)
