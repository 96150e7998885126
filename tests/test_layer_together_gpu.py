"""The layer operators as they are used: a conditioned decoder layer trained and captured, tokens
served in 8 bits, other streams, and tensors beyond 32-bit offsets."""

from __future__ import annotations

import pytest
import torch

import layer_ref as ref
from fast_mimi_amd import quantized as qz
from fast_mimi_amd import training as tr
from training_ref import assert_within

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
B, T, S, C, H, KV, D = 2, 37, 21, 128, 4, 2, 32
NAMES = ("x", "states", "w1", "qkv", "o", "w2", "q2", "kv2", "o2")


def parameters(seed, dtype, device):
    g = torch.Generator().manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g).to(device, dtype)

    return {"x": randn(B, T, C), "states": randn(B, S, C), "w1": 1 + 0.1 * randn(C), "qkv": randn(C, (H + 2 * KV) * D) * C ** -0.5,
            "o": randn(H * D, C) * C ** -0.5, "w2": 1 + 0.1 * randn(C), "q2": randn(C, H * D) * C ** -0.5,
            "kv2": randn(C, 2 * KV * D) * C ** -0.5, "o2": randn(H * D, C) * C ** -0.5}


def layer(p, freq, lengths):
    """A decoder layer that looks at an encoder's states; the last branch is added by the next norm."""
    x = p["x"]
    y = tr.rms_norm(x, p["w1"])
    qkv = (y @ p["qkv"]).view(B, T, H + 2 * KV, D)
    q, k = tr.rotary(qkv[:, :, :H], qkv[:, :, H: H + KV], freq)
    a = tr.window_attention(q, k, qkv[:, :, H + KV:], 20).reshape(B, T, H * D)
    y, h = tr.rms_norm(a @ p["o"], p["w2"], x)
    kv = (p["states"] @ p["kv2"]).view(B, S, 2 * KV, D)
    c = tr.cross_attention((y @ p["q2"]).view(B, T, H, D), kv[:, :, :KV], kv[:, :, KV:], None, lengths)
    return tr.rms_norm(c.reshape(B, T, H * D) @ p["o2"], None, h)


def plain(p, freq, lengths):
    """The same from elementary operations, in the parameters' type, on the CPU."""
    t = p["x"].dtype

    def norm(h, w=None):
        y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-5)
        return y if w is None else y * w

    def turned(z):
        angle = torch.arange(T, dtype=torch.float64)[:, None] * freq
        cos, sin = angle.cos().to(t)[:, None], angle.sin().to(t)[:, None]
        a, b = z.chunk(2, -1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    def attend(q, k, v, seen):
        k, v = k.repeat_interleave(H // KV, 2), v.repeat_interleave(H // KV, 2)
        s = (q.transpose(1, 2) @ k.permute(0, 2, 3, 1)) * D ** -0.5
        return (torch.softmax(s.masked_fill(~seen, -torch.inf), -1) @ v.transpose(1, 2)).transpose(1, 2)

    x = p["x"]
    qkv = (norm(x, p["w1"]) @ p["qkv"]).view(B, T, H + 2 * KV, D)
    i, j = torch.arange(T)[:, None], torch.arange(T)[None]
    a = attend(turned(qkv[:, :, :H]), turned(qkv[:, :, H: H + KV]), qkv[:, :, H + KV:], (j <= i) & (j > i - 20))
    h = x + a.reshape(B, T, H * D) @ p["o"]
    kv = (p["states"] @ p["kv2"]).view(B, S, 2 * KV, D)
    c = attend((norm(h, p["w2"]) @ p["q2"]).view(B, T, H, D), kv[:, :, :KV], kv[:, :, KV:],
               (torch.arange(S) < lengths[:, None])[:, None, None])
    h = h + c.reshape(B, T, H * D) @ p["o2"]
    return norm(h), h


def gradients(run, p, freq, lengths, grads):
    p = {n: v.detach().requires_grad_() for n, v in p.items()}
    out = run(p, freq, lengths)
    return [o.detach() for o in out] + list(torch.autograd.grad(out, [p[n] for n in NAMES], grads))


def test_a_layer_against_64_bits():
    """In FP32, outputs and all gradients: as near to 64 bits as elementary FP32 operations, whose roundings they
    have in other orders, but for a factor; the bounds of each operator (layer_ref) are within 8 times of
    those of their elementary forms."""
    p = parameters(1, torch.float64, "cpu")
    p = {n: v.float().double() for n, v in p.items()}
    freq, lengths = tr.rotary_frequencies(D), torch.tensor([S, 9], dtype=torch.int32)
    g = torch.Generator().manual_seed(2)
    grads = [torch.randn(B, T, C, generator=g) for _ in range(2)]
    exact = gradients(plain, p, freq, lengths, [x.double() for x in grads])
    single = gradients(plain, {n: v.float() for n, v in p.items()}, freq, lengths, grads)
    got = gradients(layer, {n: v.float().to(DEV) for n, v in p.items()}, freq.to(DEV), lengths.to(DEV), [x.to(DEV) for x in grads])
    for name, e, s, o in zip(("y", "h") + NAMES, exact, single, got):
        far, own = (o.cpu().double() - e).norm(), (s.double() - e).norm()
        assert far <= 8 * own, (name, (far / e.norm()).item(), (own / e.norm()).item())


def test_a_captured_layer():
    """Forward and backward in one graph, warmed up on a side stream: every replay gives the eager call's bits."""
    p = {n: v.requires_grad_() for n, v in parameters(3, F32, DEV).items()}
    freq, lengths = tr.rotary_frequencies(D, device=DEV), torch.tensor([S, 9], dtype=torch.int32, device=DEV)
    grads = [torch.randn(B, T, C, device=DEV) for _ in range(2)]
    leaves = [p[n] for n in NAMES]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(layer(p, freq, lengths), leaves, grads)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = layer(p, freq, lengths)
        held = [*out, *torch.autograd.grad(out, leaves, grads)]
    for seed in (4, 5, 6):
        with torch.no_grad():
            for n, v in parameters(seed, F32, DEV).items():
                p[n].copy_(v)
            lengths.copy_(torch.tensor([seed, S - seed], dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        want = gradients(layer, p, freq, lengths, grads)
        for name, a, b in zip(("y", "h") + NAMES, held, want):
            assert torch.equal(a, b), (seed, name)


@pytest.mark.parametrize("step", [
    lambda x, f: tr.rms_norm(x, None, torch.ones_like(x))[0],
    lambda x, f: tr.rotary(x, x, f)[1],
    lambda x, f: tr.cross_attention(x, x, x)])
def test_a_leaf_in_an_eager_graph_is_not_captured(step):
    x = torch.randn(2, 9, 4, 32, device=DEV, requires_grad=True)
    f = tr.rotary_frequencies(32, device=DEV)
    y = step(x, f)  # its graph stays alive
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step(x, f)
    y.backward(torch.ones_like(y))
    assert x.grad.isfinite().all()


def test_captured_functions_without_autograd():
    """Cut walks (their parts and joins), 8 bits and split products, in one graph."""
    def data(seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        return [torch.randn(shape, generator=g, device=DEV).to(BF16) for shape in ((1, 1400, 4, 64), (1, 30, 2, 64), (40, 2048))]

    kl = torch.tensor([30], dtype=torch.int32, device=DEV)
    w, ws = qz.quantize_weight(torch.randn(96, 2048, device=DEV))
    pos, freq = torch.arange(1400, device=DEV), tr.rotary_frequencies(64, device=DEV)

    def step(q, k, x):
        q, _ = tr.rotary_forward(q, None, freq, pos)
        out, lse = tr.cross_attention_forward(q, k, k, None, kl)
        grads = tr.cross_attention_backward(out, q, k, k, out, lse, None, kl)
        one, _ = tr.cross_attention_forward(k[:, :1].expand(1, 1, 2, 64).repeat(1, 1, 2, 1), q[:, :, :2], q[:, :, :2])
        x8, xs, h = qz.rms_norm(x, None, x)
        y = qz.linear(x8, xs, w, ws)
        yn, hn, rstd = tr.rms_norm_forward(x, x[0], x)
        return [out, lse, *grads, one, x8.view(torch.uint8), xs.view(torch.uint8), h, y, yn, hn,
                *tr.rms_norm_backward(yn, x, rstd, x[0], x, hn)]

    held = data(1)
    step(*held)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(*held)
    for seed in (2, 3, 4):
        for to, fresh in zip(held, data(seed)):
            to.copy_(fresh)
        kl.fill_(30 - seed)
        pos.add_(seed)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step(*held)))


def test_calls_run_on_the_current_stream():
    """Inputs made on a side stream behind slow work are what the calls there see."""
    side = torch.cuda.Stream()
    slow = torch.randn(4096, 4096, device=DEV)
    want_x = torch.randn(64, 256, generator=torch.Generator().manual_seed(1)).to(DEV)
    w, ws = qz.quantize_weight(torch.randn(64, 256, device=DEV))
    freq = tr.rotary_frequencies(64, device=DEV)
    torch.cuda.synchronize()

    def calls(x):
        q = x.view(1, 64, 4, 64)
        x8, xs = qz.quantize(x)
        return [*tr.rms_norm_forward(x, None, x), *tr.rotary_forward(q, q, freq), tr.cross_attention(q, q[:, :30], q[:, :30]),
                qz.linear(x8, xs, w, ws), qz.rms_norm(x, None, x)[2]]

    with torch.cuda.stream(side):
        x = torch.zeros(64, 256, device=DEV)
        for _ in range(20):
            slow = (slow @ slow).clamp(-1, 1)
        x.copy_(want_x)
        got = calls(x)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, calls(want_x)))


@pytest.mark.parametrize("rows", [1, 5, 16, 33, 300])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_served_projection(rows, dtype):
    """Norm to 8 bits and product: the product of the very values that the norm gave."""
    g = torch.Generator().manual_seed(rows)
    x, r = torch.randn(rows, 400, generator=g).to(BF16).to(DEV), torch.randn(rows, 400, generator=g).to(BF16).to(DEV)
    w, ws = qz.quantize_weight(torch.randn(200, 400, generator=g).to(DEV))
    stream = r
    for _ in range(2):
        x8, xs, stream = qz.rms_norm(x, None, stream)
        y = qz.linear(x8, xs, w, ws, dtype)
        want, bound = ref.product(ref.stand_for(x8, xs, 1), ref.stand_for(w, ws, 128), dtype)
        assert_within("y", y, want, bound)
        x = torch.cat((y, y), 1).to(BF16)
    assert stream.dtype == BF16


def test_a_training_loop_runs():
    """Three steps of a small model: finite gradients for every parameter at each."""
    p = {n: v.to(BF16).requires_grad_() for n, v in parameters(7, F32, DEV).items()}
    freq, lengths = tr.rotary_frequencies(D, device=DEV), torch.tensor([S, 0], dtype=torch.int32, device=DEV)
    for _ in range(3):
        y, h = layer(p, freq, lengths)
        (y.float().square().mean() + h.float().square().mean()).backward()
        for n in NAMES:
            assert torch.isfinite(p[n].grad).all() and p[n].grad.any(), n
        with torch.no_grad():
            for n in NAMES[2:]:
                p[n] -= 0.01 * p[n].grad
                p[n].grad = None
            p["x"].grad = p["states"].grad = None


def test_beyond_32_bit_offsets():
    """More than 2^31 elements: the last part as a call of its own gives it."""
    rows, c = (1 << 31) // 2048 + 5, 2048
    x = torch.empty(rows, c, dtype=BF16, device=DEV).normal_()
    y, h, rstd = tr.rms_norm_forward(x, None, x)
    for a, b in zip((y[-3:], h[-3:], rstd[-3:]), tr.rms_norm_forward(x[-3:], None, x[-3:])):
        assert torch.equal(a, b)
    dx, _, dw = tr.rms_norm_backward(y, x, rstd, None, x, h)
    assert torch.equal(dx[-3:], tr.rms_norm_backward(y[-3:], x[-3:], rstd[-3:], None, x[-3:], h[-3:])[0])
    del y, h, dx
    x8, xs = qz.quantize(x)
    for a, b in zip((x8, xs), qz.quantize(x[-3:])):
        assert torch.equal(a[-3:].view(torch.uint8), b.view(torch.uint8))
    w, ws = qz.quantize_weight(torch.randn(256, c, device=DEV))
    assert torch.equal(qz.linear(x8, xs, w, ws)[-70_000:], qz.linear(x8[-70_000:], xs[-70_000:], w, ws))
    del x8, xs
    q = x.view(1, -1, 16, 128)
    freq = tr.rotary_frequencies(128, device=DEV)
    assert torch.equal(tr.rotary_forward(q, None, freq)[0][:, -9:], tr.rotary_forward(q[:, -9:], None, freq, q.shape[1] - 9)[0])
    # Queries of two items, more than 2^31 elements before the second's end.
    q = x[: rows // 2 * 2].view(2, -1, 16, 128)
    k = torch.randn(2, 40, 16, 128, device=DEV).to(BF16)
    out, lse = tr.cross_attention_forward(q, k, k)
    dq, _, _ = tr.cross_attention_backward(q, q, k, k, out, lse)
    tail = q[1:, -64:]
    o, m = tr.cross_attention_forward(tail, k[1:], k[1:])
    val, err = ref.cross(tail, k[1:], k[1:], tail, 128 ** -0.5, None, None)
    assert_within("out", out[1:, -64:], val["out"], err["out"])
    assert_within("dq", dq[1:, -64:], val["dq"], err["dq"])
