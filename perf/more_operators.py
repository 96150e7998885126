"""What is timed: RMS norm with the residual, rotary positions, cross attention and 8-bit products, through
``fast_mimi_amd.training`` and ``fast_mimi_amd.quantized``.

Each case is a dict of plain values; ``kind`` picks the operator:

* ``norm``     RMS norm of a branch added to its residual stream, forward and backward;
* ``rotary``   rotation of queries and keys by their positions; ``train`` rotates their gradients back too;
* ``cross``    attention to the states of another sequence; ``train`` runs it forward and backward, otherwise forward only;
* ``project``  a projection as it is served: RMS norm with the residual, its output in 8 bits, their product with 8-bit weights;
* ``product``  the 8-bit product alone, of inputs that are in 8 bits already.

With ``own`` false, ``run`` computes the same from elementary torch operations in 32 bits (angles in 64), rounded once at
the end.
"""

from __future__ import annotations

import functools
import importlib
import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda:0"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-5
BLOCK = 128  # values that share a scale
FP8_MAX = 448.0


# ----------------------------------------------------------------- the cases
def listed():
    return [
        # One norm of a layer over a 1 s clip, the codec's own width: the smallest step, where launches count.
        {"name": "norm_f32_13x512", "kind": "norm", "rows": 13, "channels": 512, "type": "float32", "stream": "float32",
         "weights": "float32"},
        # A wide model in bfloat16 whose residual stream and weights stay in FP32, as mixed-precision training keeps them; an
        # odd number of rows.
        {"name": "norm_bf16_40001x4096_f32", "kind": "norm", "rows": 40_001, "channels": 4096, "type": "bfloat16",
         "stream": "float32", "weights": "float32"},
        # One token of 64 streams, each at its own far position, with frequencies stretched for long contexts; the
        # smallest call of a decoding step.
        {"name": "rotary_f16_b64_token", "kind": "rotary", "train": False, "batch": 64, "length": 1, "heads": 16, "kv_heads": 4,
         "dim": 64, "rotated": 64, "interleaved": False, "start": 1_000_000, "stretch": 16.0, "type": "float16"},
        # A training batch of packed projections, pairs side by side, half of each head rotated.
        {"name": "rotary_bf16_b8_t4095_half", "kind": "rotary", "train": True, "batch": 8, "length": 4095, "heads": 16,
         "kv_heads": 4, "dim": 128, "rotated": 64, "interleaved": True, "start": 0, "stretch": 1.0, "type": "bfloat16"},
        # A layer over a 1 s clip that looks at a short prompt, in FP32.
        {"name": "cross_f32_b1_t13_s7", "kind": "cross", "train": True, "batch": 1, "queries": 13, "keys": 7, "heads": 8,
         "kv_heads": 8, "dim": 64, "padded": False, "type": "float32"},
        # Eight clips of 100 s over texts of up to 300 tokens: many queries, few keys, both padded.
        {"name": "cross_bf16_b8_t2500_s300_padded", "kind": "cross", "train": True, "batch": 8, "queries": 2500, "keys": 300,
         "heads": 8, "kv_heads": 8, "dim": 64, "padded": True, "type": "bfloat16"},
        # Long clips over the states of an encoder as long as they are, four query heads to a key head.
        {"name": "cross_bf16_b2_t4095_s4001_gqa", "kind": "cross", "train": True, "batch": 2, "queries": 4095, "keys": 4001,
         "heads": 16, "kv_heads": 4, "dim": 128, "padded": False, "type": "bfloat16"},
        # One new token of 8 streams over an encoder's states, forward only.
        {"name": "cross_f16_b8_token_s8000", "kind": "cross", "train": False, "batch": 8, "queries": 1, "keys": 8000, "heads": 16,
         "kv_heads": 4, "dim": 64, "padded": False, "type": "float16"},
        # One new token through a projection: the weights' bytes count.
        {"name": "project_bf16_1x4096_to_6144", "kind": "project", "rows": 1, "channels": 4096, "out": 6144, "type": "bfloat16"},
        # A 10 s batch of 8 clips through a feed-forward projection; an odd number of rows.
        {"name": "project_bf16_1001x2048_to_8192", "kind": "project", "rows": 1001, "channels": 2048, "out": 8192,
         "type": "bfloat16"},
        # 32 streams' tokens through the projection back.
        {"name": "product_bf16_32x8192_to_2048", "kind": "product", "rows": 32, "channels": 8192, "out": 2048, "type": "bfloat16"},
        # Long prompts of a batch through a wide projection: the largest product.
        {"name": "product_bf16_8192x8192_to_8192", "kind": "product", "rows": 8192, "channels": 8192, "out": 8192,
         "type": "bfloat16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["norm", "rotary", "cross", "cross", "project", "product"])
    case = {"kind": kind, "type": rng.choice(sorted(TYPES))}
    if kind == "norm":
        channels = rng.choice([64, 257, 512, 768, 1000, 1024, 2047, 2048, 4096, 8192])
        return {**case, "rows": _log(rng, 1, min(160_000, 40_000 * 4096 // channels)), "channels": channels,
                "stream": rng.choice([case["type"], "float32"]), "weights": rng.choice([case["type"], "float32"])}
    if kind == "rotary":
        kv_heads = rng.choice([1, 2, 4, 8])
        dim = rng.choice([32, 64, 80, 96, 128, 128])
        batch = _log(rng, 1, 64)
        heads = kv_heads * rng.choice([1, 2, 4])
        length = _log(rng, 1, max(1, min(8192, 8 * 4095 * 20 * 128 // 2 // (batch * (heads + kv_heads) * dim))))
        return {**case, "train": rng.random() < 0.5, "batch": batch, "length": length, "heads": heads, "kv_heads": kv_heads,
                "dim": dim, "rotated": rng.choice([dim, dim, dim // 2]), "interleaved": rng.random() < 0.5,
                "start": rng.choice([0, 0, 5000, 1_000_000]), "stretch": rng.choice([1.0, 1.0, 4.0, 16.0])}
    if kind in ("project", "product"):
        channels = 16 * _log(rng, 4, 512)
        if rng.random() < 0.5:
            channels = max(BLOCK, channels // BLOCK * BLOCK)
        if kind == "project":  # served in 16 bits: an FP32 activation would say little behind an input of four bits
            case["type"] = rng.choice(["bfloat16", "float16"])
        out = _log(rng, 64, 8192)
        if rng.random() < 0.7:
            out = (out + 15) // 16 * 16
        return {**case, "rows": _log(rng, 1, 8192), "channels": channels, "out": out}
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    case.update(heads=heads, kv_heads=kv_heads, dim=rng.choice([32, 64, 64, 128]), padded=rng.random() < 0.4)
    batch = _log(rng, 1, 16)
    if rng.random() < 0.25:
        return {**case, "train": False, "batch": batch, "queries": rng.choice([1, 1, 2, 5]), "keys": _log(rng, 1, 8000)}
    # The plain form keeps batch x heads x queries x keys scores; FP32 pairs cost more than 16-bit ones.
    pairs = (100_000_000 if case["type"] == "float32" else 400_000_000) // (batch * heads)
    queries = _log(rng, 1, min(4096, pairs))
    return {**case, "train": True, "batch": batch, "queries": queries, "keys": _log(rng, 1, min(4096, pairs // queries))}


# ------------------------------------------------------------------- inputs
def _exponents(amax):
    """The least e with amax <= 448 * 2^e (a block of zeros: 0), within what a scale of one byte holds."""
    m, x = torch.frexp(amax)
    e = x - 9 + (m > FP8_MAX / 512).to(x.dtype)
    return torch.where(amax == 0, torch.zeros_like(e), e).clamp(-127, 127)


def _blocks(x, rows):
    """x [R, C], padded by zeros to whole blocks of `rows` x 128 values, as [R / rows, rows, C / 128, 128]."""
    r, c = x.shape
    x = torch.nn.functional.pad(x, (0, -c % BLOCK, 0, -r % rows))
    return x.reshape(x.shape[0] // rows, rows, x.shape[1] // BLOCK, BLOCK)


def _in_8_bits(x, rows):
    """(values in e4m3, scales in e8m0 [R / rows, C / 128]) of FP32 x [R, C]; `rows` rows share a scale."""
    r, c = x.shape
    blocks = _blocks(x, rows)
    e = _exponents(blocks.abs().amax((1, 3)))
    q = blocks * torch.exp2(-e.float())[:, None, :, None]
    q = q.reshape(blocks.shape[0] * rows, -1)[:r, :c].contiguous().to(torch.float8_e4m3fn)
    return q, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dtype = TYPES[case["type"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    def stream(rows, c):
        # A residual stream: rows of their own scale, a few large channels.
        x = randn(rows, c) * (0.5 + torch.rand((rows, 1), generator=g, device=DEV))
        x[:, :: max(1, c // 3)] *= 4
        return x

    if case["kind"] == "norm":
        rows, c, st = case["rows"], case["channels"], TYPES[case["stream"]]
        return {"case": case, "x": (0.5 * randn(rows, c)).to(dtype), "residual": stream(rows, c).to(st),
                "weight": (1 + 0.1 * randn(c)).to(TYPES[case["weights"]]), "grad": randn(rows, c).to(dtype),
                "grad_h": randn(rows, c).to(st)}
    if case["kind"] == "rotary":
        b, t, h, kv, d = (case[n] for n in ("batch", "length", "heads", "kv_heads", "dim"))
        half = case["rotated"] // 2
        freq = 10_000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
        # Stretched contexts: the slow half of the frequencies is slower by the factor.
        freq = torch.where(torch.arange(half, device=DEV) >= half // 2, freq / case["stretch"], freq)
        positions = torch.arange(t, device=DEV).expand(b, t)
        if case["start"]:
            positions = positions + torch.randint(0, case["start"], (b, 1), generator=g, device=DEV)
        state = {"case": case, "frequencies": freq, "positions": positions.contiguous(),
                 "scale": 1 + 0.1 * math.log(case["stretch"])}
        # One packed projection, as the transformer layers make it.
        qkv = randn(b, t, (h + 2 * kv) * d).to(dtype)
        state["q"] = qkv[..., : h * d].view(b, t, h, d)
        state["k"] = qkv[..., h * d: (h + kv) * d].view(b, t, kv, d)
        if case["train"]:
            state["dq"], state["dk"] = randn(b, t, h, d).to(dtype), randn(b, t, kv, d).to(dtype)
        return state
    if case["kind"] in ("project", "product"):
        rows, c, n = case["rows"], case["channels"], case["out"]
        w = randn(n, c) * (0.5 + torch.rand((n, 1), generator=g, device=DEV)) * c ** -0.5
        state = {"case": case, "dtype": dtype}
        state["w"], state["w_scale"] = _in_8_bits(w, BLOCK)
        if case["kind"] == "product":
            state["x"], state["x_scale"] = _in_8_bits(stream(rows, c), 1)
        else:
            state.update(x=(0.5 * randn(rows, c)).to(dtype), residual=stream(rows, c).to(dtype), weight=(1 + 0.1 * randn(c)).to(dtype))
        return state
    b, t, s, h, kv, d = (case[n] for n in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    state = {"case": case, "scale": d ** -0.5, "key_lengths": None, "query_lengths": None}
    if case["padded"]:
        # Texts of all lengths, the first of them whole and the last one, in larger batches, empty (a dropped condition).
        lengths = torch.randint(1, s + 1, (b,), generator=g, device=DEV)
        lengths[0] = s
        if b >= 4:
            lengths[-1] = 0
        state["key_lengths"] = lengths.to(torch.int32)
        short = torch.randint(1, t + 1, (b,), generator=g, device=DEV)
        state["query_lengths"] = torch.where(torch.arange(b, device=DEV) % 4 == 1, short, t).to(torch.int32)
    # The encoder's states are projected to keys and values in one.
    kv_packed = randn(b, s, 2 * kv * d).to(dtype)
    state.update(q=(1.5 * randn(b, t, h, d)).to(dtype), k=kv_packed[..., : kv * d].view(b, s, kv, d),
                 v=kv_packed[..., kv * d:].view(b, s, kv, d))
    if case["train"]:
        state["grad"] = randn(b, t, h, d).to(dtype)
    return state


# ------------------------------------------------------------ one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"norm": _own_norm, "rotary": _own_rotary, "cross": _own_cross, "project": _own_project,
                "product": _own_product}[kind](state)
    return {"norm": _norm, "rotary": _rotary, "cross": _cross, "project": _project, "product": _product}[kind](state)


@functools.lru_cache(maxsize=None)
def _own(name):
    path = str(Path(__file__).resolve().parents[1] / "fast-mimi_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    return importlib.import_module("fast_mimi_amd." + name)


def _own_norm(state):
    f = _own("training")
    y, h, rstd = f.rms_norm_forward(state["x"], state["weight"], state["residual"], EPS)
    # What a program keeps for the backward pass: an FP32 stream's sum, or the two 16-bit parts of it.
    x, residual = (h, None) if h.dtype == torch.float32 else (state["x"], state["residual"])
    dx, dh, dw = f.rms_norm_backward(state["grad"], x, rstd, state["weight"], residual, state["grad_h"])
    return {"y": y, "h": h, "dx": dx, "dresidual": dh, "dw": dw}


def _own_rotary(state):
    f, how = _own("training"), (state["frequencies"], state["positions"], state["case"]["interleaved"], state["scale"])
    q, k = f.rotary_forward(state["q"], state["k"], *how)
    if not state["case"]["train"]:
        return {"q": q, "k": k}
    dq, dk = f.rotary_backward(state["dq"], state["dk"], *how)
    return {"q": q, "k": k, "dq": dq, "dk": dk}


def _own_cross(state):
    f, q, k, v = _own("training"), state["q"], state["k"], state["v"]
    how = {"scale": state["scale"], "key_lengths": state["key_lengths"], "query_lengths": state["query_lengths"]}
    out, lse = f.cross_attention_forward(q, k, v, **how)
    if not state["case"]["train"]:
        return {"out": out}
    dq, dk, dv = f.cross_attention_backward(state["grad"], q, k, v, out, lse, **how)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _own_project(state):
    f = _own("quantized")
    x, x_scale, h = f.rms_norm(state["x"], state["weight"], state["residual"], EPS)
    return {"y": f.linear(x, x_scale, state["w"], state["w_scale"], state["dtype"]), "h": h}


def _own_product(state):
    return {"y": _own("quantized").linear(state["x"], state["x_scale"], state["w"], state["w_scale"], state["dtype"])}


def _norm(state):
    w, grad = state["weight"].float(), state["grad"].float()
    h = state["x"].float() + state["residual"].float()
    rstd = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
    hh = h * rstd
    g = grad * w
    dh = state["grad_h"].float() + rstd * (g - hh * (g * hh).mean(1, keepdim=True))
    t, st = state["x"].dtype, state["residual"].dtype
    return {"y": (hh * w).to(t), "h": h.to(st), "dx": dh.to(t), "dresidual": dh.to(st),
            "dw": (grad * hh).sum(0).to(state["weight"].dtype)}


def _turned(x, cos, sin, rotated, interleaved):
    """x [B, T, H, D] with its first `rotated` channels turned by the angles of cos, sin [B, T, 1, rotated / 2]."""
    y = x.float()
    part = y[..., :rotated]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else part.chunk(2, -1)
    turned = (a * cos - b * sin, b * cos + a * sin)
    part = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return torch.cat((part, y[..., rotated:]), -1).to(x.dtype)


def _rotary(state):
    case = state["case"]
    angle = state["positions"].double()[..., None] * state["frequencies"]
    cos = (torch.cos(angle) * state["scale"]).float()[:, :, None]
    sin = (torch.sin(angle) * state["scale"]).float()[:, :, None]
    how = case["rotated"], case["interleaved"]
    out = {"q": _turned(state["q"], cos, sin, *how), "k": _turned(state["k"], cos, sin, *how)}
    if case["train"]:
        out.update(dq=_turned(state["dq"], cos, -sin, *how), dk=_turned(state["dk"], cos, -sin, *how))
    return out


def _cross(state):
    case, dtype = state["case"], state["q"].dtype
    b, t, s, h, kv, d = (case[n] for n in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    n = h // kv

    def rows(x):  # [B, T, H, D] -> [B, KV, n * T, D]: the query heads of a key head together
        return x.float().reshape(b, t, kv, n, d).permute(0, 2, 3, 1, 4).reshape(b, kv, n * t, d)

    def back(x):
        return x.reshape(b, kv, n, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, h, d).to(dtype)

    q, k, v = rows(state["q"]), state["k"].float().transpose(1, 2), state["v"].float().transpose(1, 2)
    score = (q @ k.transpose(2, 3).contiguous()).mul_(state["scale"])
    if state["key_lengths"] is not None:
        seen = torch.arange(s, device=DEV) < state["key_lengths"][:, None]
        there = torch.arange(t, device=DEV) < state["query_lengths"][:, None]
        seen = (seen[:, None] & there[:, :, None])[:, None, None].expand(b, 1, n, t, s).reshape(b, 1, n * t, s)
        score.masked_fill_(~seen, -math.inf)
    top = score.amax(3, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(3, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total))
    out = p @ v
    if not case["train"]:
        return {"out": back(out)}
    # Padded queries see nothing: their probabilities, and so their gradients, are zeros.
    grad = rows(state["grad"])
    dv = p.transpose(2, 3) @ grad
    dp = grad @ v.transpose(2, 3).contiguous()
    ds = dp.sub_((grad * out).sum(3, keepdim=True)).mul_(p)
    dq, dk = (ds @ k) * state["scale"], (ds.transpose(2, 3) @ q) * state["scale"]
    return {"out": back(out), "dq": back(dq), "dk": dk.transpose(1, 2).contiguous().to(dtype),
            "dv": dv.transpose(1, 2).contiguous().to(dtype)}


def _scaled(x, scale, rows):
    """The FP32 values that e4m3 x [R, C] and its scales stand for."""
    r, c = x.shape
    s = torch.exp2(scale.view(torch.uint8).float() - 127)
    return (_blocks(x.float(), rows) * s[:, None, :, None]).reshape(s.shape[0] * rows, -1)[:r, :c]


def _product(state):
    y = _scaled(state["x"], state["x_scale"], 1) @ _scaled(state["w"], state["w_scale"], BLOCK).t()
    return {"y": y.to(state["dtype"])}


def _project(state):
    h = state["x"].float() + state["residual"].float()
    y = h * (1 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)) * state["weight"].float()
    x, x_scale = _in_8_bits(y, 1)
    return {**_product({**state, "x": x, "x_scale": x_scale}), "h": h.to(state["residual"].dtype)}


# --------------------------------------------------- from the definition, in 64 bits
def _exact_8_bits(y):
    """The values that blocks of 128 of float64 rows y [R, C] stand for in e4m3 with their power of two: the nearest of the
    format's values, ties to the even one."""
    out = torch.empty_like(y)
    for first in range(0, y.shape[1], BLOCK):
        part = y[:, first: first + BLOCK]
        most = part.abs().amax(1, keepdim=True)
        e = torch.ceil(torch.log2(torch.where(most == 0, 1.0, most) / FP8_MAX))
        e = torch.where(most > FP8_MAX * torch.exp2(e), e + 1, torch.where(most <= FP8_MAX * torch.exp2(e - 1), e - 1, e))
        v = part / torch.exp2(e)
        size = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
        step = torch.exp2(size - 3)
        out[:, first: first + BLOCK] = torch.round(v / step) * step * torch.exp2(e)
    return out


def _exact_weights(w, scale):
    exponent = scale.view(torch.uint8).double() - 127
    full = exponent.repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)[: w.shape[0], : w.shape[1]]
    return w.double() * torch.exp2(full)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "norm":
        x, r, w = (state[n].double().requires_grad_() for n in ("x", "residual", "weight"))
        h = x + r
        y = h / torch.sqrt(h.square().mean(1, keepdim=True) + EPS) * w
        dx, dr, dw = torch.autograd.grad((y, h), (x, r, w), (state["grad"].double(), state["grad_h"].double()))
        return {"y": y.detach(), "h": h.detach(), "dx": dx, "dresidual": dr, "dw": dw}
    if case["kind"] == "rotary":
        half = case["rotated"] // 2
        turn = torch.polar(torch.full((), state["scale"], dtype=torch.float64, device=DEV),
                           state["positions"].double()[:, :, None, None] * state["frequencies"])

        def rotate(x, by):
            x = x.double()
            part = x[..., : 2 * half]
            part = part.unflatten(-1, (half, 2)) if case["interleaved"] else part.unflatten(-1, (2, half)).transpose(-1, -2)
            part = torch.view_as_real(torch.view_as_complex(part.contiguous()) * by)
            part = part if case["interleaved"] else part.transpose(-1, -2)
            return torch.cat((part.flatten(-2), x[..., 2 * half:]), -1)

        out = {"q": rotate(state["q"], turn), "k": rotate(state["k"], turn)}
        if case["train"]:
            out.update(dq=rotate(state["dq"], turn.conj()), dk=rotate(state["dk"], turn.conj()))
        return out
    if case["kind"] in ("project", "product"):
        w = _exact_weights(state["w"], state["w_scale"])
        if case["kind"] == "product":
            exponent = (state["x_scale"].view(torch.uint8).double() - 127).repeat_interleave(BLOCK, 1)[:, : case["channels"]]
            return {"y": (state["x"].double() * torch.exp2(exponent)) @ w.t()}
        h = state["x"].double() + state["residual"].double()
        x = _exact_8_bits(h / torch.sqrt(h.square().mean(1, keepdim=True) + EPS) * state["weight"].double())
        return {"y": x @ w.t(), "h": h}
    # Softmax attention and its derivative, one clip and key head at a time, over its valid positions only.
    t, s, n = case["queries"], case["keys"], case["heads"] // case["kv_heads"]
    names = ("q", "k", "v")
    full = {m: torch.zeros(state[m].shape, dtype=torch.float64, device=DEV) for m in names}
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device=DEV)
    for b in range(case["batch"]):
        rows = t if state["query_lengths"] is None else int(state["query_lengths"][b])
        keys = s if state["key_lengths"] is None else int(state["key_lengths"][b])
        if rows == 0 or keys == 0:
            continue
        for a in range(case["kv_heads"]):
            heads = slice(a * n, (a + 1) * n)
            leaf = (state["q"][b, :rows, heads], state["k"][b, :keys, a], state["v"][b, :keys, a])
            q, k, v = (x.double().requires_grad_(case["train"]) for x in leaf)
            o = torch.softmax(torch.einsum("thd,sd->hts", q, k) * state["scale"], 2) @ v
            o = o.transpose(0, 1)
            out[b, :rows, heads] = o.detach()
            if case["train"]:
                dq, dk, dv = torch.autograd.grad(o, (q, k, v), state["grad"][b, :rows, heads].double())
                full["q"][b, :rows, heads], full["k"][b, :keys, a], full["v"][b, :keys, a] = dq, dk, dv
    return {"out": out, **({"d" + m: full[m] for m in names} if case["train"] else {})}


# ------------------------------------------------------------------ the floor
def work(case):
    size = 4 if case["type"] == "float32" else 2
    if case["kind"] == "norm":
        n, st = case["rows"] * case["channels"], 4 if case["stream"] == "float32" else 2
        # x, the stream, dy and the stream's gradient in; y, the stream and its gradient, and dx where that is of another
        # type, out; h once more for the backward pass.
        out = 2 * size if st != size else size
        return {"bytes": n * (2 * size + 4 * st + out) + 2 * case["channels"] * (4 if case["weights"] == "float32" else 2),
                "flops": 14 * n}
    if case["kind"] == "rotary":
        n = case["batch"] * case["length"] * (case["heads"] + case["kv_heads"])
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2 * n * case["dim"] * size + 8 * case["batch"] * case["length"]),
                "flops": passes * 3 * n * case["rotated"]}
    if case["kind"] in ("project", "product"):
        rows, c, n = case["rows"], case["channels"], case["out"]
        inputs = 3 * rows * c * size if case["kind"] == "project" else rows * c
        return {"bytes": inputs + n * c + rows * n * size, "flops": 2 * rows * c * n}
    b, t, s, h, kv, d = (case[n] for n in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    passes = 2 if case["train"] else 1  # q, out and k, v; with gradients dout, dq and dk, dv
    # Forward two products; backward five, one of them the scores again.
    return {"bytes": passes * size * b * d * (2 * h * t + 2 * kv * s), "flops": (14 if case["train"] else 4) * d * b * h * t * s}
