"""What is timed: the training operators, through ``fast_mimi_amd.training``.

Each case is a dict of plain values; ``kind`` picks the operator:

* ``norm``    LayerNorm over the channels, forward and backward (input, weight and bias gradients);
* ``attend``  causal sliding-window attention of projected queries, keys and values: ``train`` runs it forward and
              backward, otherwise it runs forward only (a single token over the frames before it);
* ``embed``   the sum of a frame's codebook entries, forward and backward (the gradient of every codebook).

With ``own`` false, ``run`` computes the same from elementary torch operations in 32 bits, rounded once at the end.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-5
ENTRIES = 2048


# ----------------------------------------------------------------- the cases
def listed():
    return [
        # One LayerNorm of a transformer over a 1 s clip: the smallest step, where launches count.
        {"name": "norm_f32_13x512", "kind": "norm", "rows": 13, "channels": 512, "type": "float32", "weights": "float32"},
        # A wider trunk in bfloat16 with FP32 weights, as mixed-precision training keeps them; an odd number of rows.
        {"name": "norm_bf16_8191x2048", "kind": "norm", "rows": 8191, "channels": 2048, "type": "bfloat16",
         "weights": "float32"},
        # 64 clips of 100 s: the largest batch one GPU trains on.
        {"name": "norm_f32_160000x512", "kind": "norm", "rows": 160_000, "channels": 512, "type": "float32",
         "weights": "float32"},
        # Attention of one layer over a 1 s clip.
        {"name": "attend_f32_b1_t13", "kind": "attend", "train": True, "batch": 1, "queries": 13, "keys": 13, "heads": 8,
         "kv_heads": 8, "dim": 64, "window": 250, "padded": False, "type": "float32"},
        # A training batch of 16 clips of up to 10 s, a quarter of them shorter and padded.
        {"name": "attend_f32_b16_t250_padded", "kind": "attend", "train": True, "batch": 16, "queries": 250, "keys": 250,
         "heads": 8, "kv_heads": 8, "dim": 64, "window": 250, "padded": True, "type": "float32"},
        # One 100 s clip in bfloat16: ten windows long.
        {"name": "attend_bf16_b1_t2500", "kind": "attend", "train": True, "batch": 1, "queries": 2500, "keys": 2500,
         "heads": 8, "kv_heads": 8, "dim": 64, "window": 250, "padded": False, "type": "bfloat16"},
        # 16 clips of 100 s in FP32, the codec's own precision.
        {"name": "attend_f32_b16_t2500", "kind": "attend", "train": True, "batch": 16, "queries": 2500, "keys": 2500,
         "heads": 8, "kv_heads": 8, "dim": 64, "window": 250, "padded": False, "type": "float32"},
        # A transformer over the codes without a window, four query heads to a key head, an odd length.
        {"name": "attend_bf16_b2_t4095_gqa", "kind": "attend", "train": True, "batch": 2, "queries": 4095, "keys": 4095,
         "heads": 16, "kv_heads": 4, "dim": 128, "window": 0, "padded": False, "type": "bfloat16"},
        # One new token of 8 streams over all positions that the model has, forward only.
        {"name": "attend_f16_b8_token_8000", "kind": "attend", "train": False, "batch": 8, "queries": 1, "keys": 8000,
         "heads": 16, "kv_heads": 4, "dim": 64, "window": 0, "padded": False, "type": "float16"},
        # The codebook sum of a 1 s clip.
        {"name": "embed_f32_b1_q8_t13", "kind": "embed", "batch": 1, "books": 8, "frames": 13, "dim": 256,
         "skew": False, "type": "float32"},
        # 64 clips of 10 s with all 32 codebooks.
        {"name": "embed_f32_b64_q32_t125", "kind": "embed", "batch": 64, "books": 32, "frames": 125, "dim": 256,
         "skew": False, "type": "float32"},
        # Wide embeddings of long clips in bfloat16; a third of the frames are silence, which is one code, and the
        # shorter clips are padded.
        {"name": "embed_bf16_b16_q8_t1500_skew", "kind": "embed", "batch": 16, "books": 8, "frames": 1500, "dim": 1024,
         "skew": True, "type": "bfloat16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["norm", "attend", "attend", "embed"])
    case = {"kind": kind, "type": rng.choice(sorted(TYPES))}
    if kind == "norm":
        channels = rng.choice([64, 256, 512, 513, 768, 1000, 1024, 2047, 2048, 4096])
        return {**case, "rows": _log(rng, 1, min(200_000, 160_000 * 512 // channels)), "channels": channels,
                "weights": rng.choice([case["type"], "float32"])}
    if kind == "embed":
        dim = rng.choice([64, 200, 256, 512, 1024])
        books = rng.choice([1, 2, 4, 8, 16, 32])
        while books * dim > 8192:
            books //= 2
        batch = _log(rng, 1, 64)
        frames = _log(rng, 1, max(1, min(6000, 24_000 * 8192 // (books * dim * batch), 60_000 // batch)))
        return {**case, "batch": batch, "books": books, "frames": frames, "dim": dim, "skew": rng.random() < 0.5}
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    case.update(heads=heads, kv_heads=kv_heads, dim=rng.choice([32, 64, 64, 128]), padded=rng.random() < 0.3)
    if rng.random() < 0.25:
        batch = _log(rng, 1, 16)
        return {**case, "train": False, "batch": batch, "queries": rng.choice([1, 1, 2, 5]),
                "keys": _log(rng, 8, 8000), "window": rng.choice([0, 0, 250])}
    batch = _log(rng, 1, 16)
    # The plain form keeps batch x heads x keys^2 scores; FP32 pairs cost more than 16-bit ones.
    top = math.isqrt(200_000_000 // (batch * heads) if case["type"] == "float32" else 400_000_000 // (batch * heads))
    keys = _log(rng, 2, min(4096, top))
    queries = keys if rng.random() < 0.7 else rng.randint(1, keys)
    return {**case, "train": True, "batch": batch, "queries": queries, "keys": keys,
            "window": rng.choice([0, 100, 250, 250, 777])}


# ------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dtype = TYPES[case["type"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    if case["kind"] == "norm":
        rows, c, wt = case["rows"], case["channels"], TYPES[case["weights"]]
        # A residual stream: rows of their own scale around a common offset, a few large channels.
        x = randn(rows, c) * (0.5 + torch.rand((rows, 1), generator=g, device=DEV)) + 0.3 * randn(c)
        x[:, :: max(1, c // 3)] *= 4
        return {"case": case, "x": x.to(dtype), "grad": randn(rows, c).to(dtype),
                "weight": (1 + 0.1 * randn(c)).to(wt), "bias": (0.1 * randn(c)).to(wt)}
    if case["kind"] == "embed":
        b, q, t, d = case["batch"], case["books"], case["frames"], case["dim"]
        codes = torch.randint(0, ENTRIES, (b, q, t), generator=g, device=DEV)
        if case["skew"]:
            silent = torch.rand((b, 1, t), generator=g, device=DEV) < 1 / 3
            codes = torch.where(silent, torch.arange(7, 7 + q, device=DEV)[None, :, None], codes)
            if b >= 4:
                codes[b - b // 4:, :, max(1, int(0.6 * t)):] = -1  # padding
        return {"case": case, "codes": codes, "table": (0.02 * randn(q, ENTRIES, d)).to(dtype),
                "grad": randn(b, t, d).to(dtype), "scale": math.sqrt(d)}
    b, t, s, h, kv, d = (case[n] for n in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    lengths = None
    if case["padded"]:
        # Every fourth clip is shorter.
        short = torch.randint(1, s + 1, (b,), generator=g, device=DEV)
        lengths = torch.where(torch.arange(b, device=DEV) % 4 == 3, short, s).to(torch.int32)
    state = {"case": case, "lengths": lengths, "window": case["window"] or None, "scale": d ** -0.5}
    if t == s:
        # One packed projection, as the transformer layers make it.
        qkv = randn(b, t, (h + 2 * kv) * d)
        qkv[..., : h * d] *= 1.5
        qkv = qkv.to(dtype)
        state["q"] = qkv[..., : h * d].view(b, t, h, d)
        state["k"] = qkv[..., h * d: (h + kv) * d].view(b, s, kv, d)
        state["v"] = qkv[..., (h + kv) * d:].view(b, s, kv, d)
    else:
        # A cache of keys and values, the queries of its last positions.
        state.update(q=(1.5 * randn(b, t, h, d)).to(dtype), k=randn(b, s, kv, d).to(dtype), v=randn(b, s, kv, d).to(dtype))
    if case["train"]:
        state["grad"] = randn(b, t, h, d).to(dtype)
    return state


def _visible(case, lengths):
    """[B or 1, T, S]: key j of a clip is visible from the query at position p iff p - window < j <= p < length."""
    s, t, w = case["keys"], case["queries"], case["window"]
    p = torch.arange(s - t, s, device=DEV)[:, None]
    j = torch.arange(s, device=DEV)[None, :]
    seen = j <= p
    if w:
        seen = seen & (j > p - w)
    seen = seen[None]
    return seen if lengths is None else seen & (p[None] < lengths[:, None, None])


# ------------------------------------------------------------ one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"norm": _own_norm, "attend": _own_attend, "embed": _own_embed}[kind](state)
    return {"norm": _norm, "attend": _attend, "embed": _embed}[kind](state)


def _own():
    import sys
    from pathlib import Path

    path = str(Path(__file__).resolve().parents[1] / "fast-mimi_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from fast_mimi_amd import training

    return training


def _own_norm(state):
    f, x, w, b = _own(), state["x"], state["weight"], state["bias"]
    y, mean, rstd = f.layer_norm_forward(x, w, b, EPS)
    dx, dw, db = f.layer_norm_backward(state["grad"], x, mean, rstd, w, b)
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def _own_attend(state):
    f, q, k, v = _own(), state["q"], state["k"], state["v"]
    how = {"window": state["window"], "scale": state["scale"], "lengths": state["lengths"]}
    out, lse = f.window_attention_forward(q, k, v, **how)
    if not state["case"]["train"]:
        return {"out": out}
    dq, dk, dv = f.window_attention_backward(state["grad"], q, k, v, out, lse, **how)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _own_embed(state):
    f, codes, table, scale = _own(), state["codes"], state["table"], state["scale"]
    out = f.code_embedding_forward(codes, table, scale)
    return {"out": out, "dtable": f.code_embedding_backward(state["grad"], codes, table, scale)}


def _norm(state):
    x, grad, w = state["x"].float(), state["grad"].float(), state["weight"].float()
    d = x - x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    xh = d * rstd
    g = grad * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    wt = state["weight"].dtype
    return {"y": (xh * w + state["bias"].float()).to(state["x"].dtype), "dx": dx.to(state["x"].dtype),
            "dw": (grad * xh).sum(0).to(wt), "db": grad.sum(0).to(wt)}


def _attend(state):
    case, dtype = state["case"], state["q"].dtype
    b, t, s, h, kv, d = (case[n] for n in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    n = h // kv

    def rows(x):  # [B, T, H, D] -> [B, KV, n * T, D]: the query heads of a key head together
        return x.float().reshape(b, t, kv, n, d).permute(0, 2, 3, 1, 4).reshape(b, kv, n * t, d)

    def back(x):
        return x.reshape(b, kv, n, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, h, d).to(dtype)

    q, k, v = rows(state["q"]), state["k"].float().transpose(1, 2), state["v"].float().transpose(1, 2)
    seen = _visible(case, state["lengths"])[:, None, None].expand(-1, 1, n, t, s).reshape(-1, 1, n * t, s)
    score = (q @ k.transpose(2, 3).contiguous()).mul_(state["scale"]).masked_fill_(~seen, -math.inf)
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


def _embed(state):
    codes, table, scale = state["codes"], state["table"], state["scale"]
    books, entries, dim = table.shape
    there = (codes >= 0)[..., None]
    at = codes.clamp(min=0) + entries * torch.arange(books, device=DEV)[None, :, None]
    flat = table.reshape(books * entries, dim)
    out = (flat[at].float() * there).sum(1) * scale
    grad = (state["grad"].float()[:, None] * there).reshape(-1, dim)
    dtable = torch.zeros((books * entries, dim), device=DEV).index_add_(0, at.reshape(-1), grad) * scale
    return {"out": out.to(table.dtype), "dtable": dtable.reshape(table.shape).to(table.dtype)}


# --------------------------------------------------- from the definition, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "norm":
        x, w, b = (state[n].double().requires_grad_() for n in ("x", "weight", "bias"))
        y = torch.nn.functional.layer_norm(x, (case["channels"],), w, b, EPS)
        return dict(zip(("y", "dx", "dw", "db"), (y.detach(), *torch.autograd.grad(y, (x, w, b), state["grad"].double()))))
    if case["kind"] == "embed":
        codes, books = state["codes"], case["books"]
        table = state["table"].double()
        out = torch.zeros((case["batch"], case["frames"], case["dim"]), dtype=torch.float64, device=DEV)
        dtable, grad = torch.zeros_like(table), state["grad"].double()
        for j in range(books):
            where = codes[:, j] >= 0
            out[where] += table[j][codes[:, j][where]]
            dtable[j].index_put_((codes[:, j][where],), grad[where], accumulate=True)
        return {"out": out * state["scale"], "dtable": dtable * state["scale"]}
    # Softmax attention and its derivative, one clip and key head at a time, over its valid positions only.
    t, s, w, n = case["queries"], case["keys"], case["window"], case["heads"] // case["kv_heads"]
    names = ("q", "k", "v")
    full = {m: torch.zeros(state[m].shape, dtype=torch.float64, device=DEV) for m in names}
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device=DEV)
    p, j = torch.arange(s - t, s, device=DEV)[:, None], torch.arange(s, device=DEV)[None]
    hidden = (j > p) if not w else (j > p) | (j <= p - w)
    for b in range(case["batch"]):
        length = s if state["lengths"] is None else int(state["lengths"][b])
        rows = max(0, length - (s - t))
        if rows == 0:
            continue
        for a in range(case["kv_heads"]):
            heads = slice(a * n, (a + 1) * n)
            leaf = (state["q"][b, :rows, heads], state["k"][b, :length, a], state["v"][b, :length, a])
            q, k, v = (x.double().requires_grad_(case["train"]) for x in leaf)
            score = torch.einsum("thd,sd->hts", q, k) * state["scale"]
            o = torch.softmax(score.masked_fill(hidden[:rows, :length], -math.inf), 2) @ v
            o = o.transpose(0, 1)
            out[b, :rows, heads] = o.detach()
            if case["train"]:
                dq, dk, dv = torch.autograd.grad(o, (q, k, v), state["grad"][b, :rows, heads].double())
                full["q"][b, :rows, heads], full["k"][b, :length, a], full["v"][b, :length, a] = dq, dk, dv
    return {"out": out, **({"d" + m: full[m] for m in names} if case["train"] else {})}


# ------------------------------------------------------------------ the floor
def _pairs(case):
    """Visible (query, key) pairs of one clip and head, without padding."""
    s, t, w = case["keys"], case["queries"], case["window"] or case["keys"]
    return sum(min(p + 1, w) for p in range(s - t, s))


def work(case):
    size = 4 if case["type"] == "float32" else 2
    if case["kind"] == "norm":
        n = case["rows"] * case["channels"]
        # x and dy in, y and dx out; two flops each for the centring, the square, the affine and six products behind.
        return {"bytes": 4 * n * size + 4 * case["channels"] * (4 if case["weights"] == "float32" else 2), "flops": 20 * n}
    if case["kind"] == "embed":
        rows, n = case["batch"] * case["frames"], case["books"] * ENTRIES * case["dim"]
        read = min(n, rows * case["books"] * case["dim"])  # the entries that are named
        return {"bytes": 8 * rows * case["books"] + size * (2 * rows * case["dim"] + read + n),
                "flops": 2 * rows * case["books"] * case["dim"]}
    b, t, s, h, kv, d = (case[n] for n in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    pairs = b * h * _pairs(case)
    near = min(s, (case["window"] or s) + t - 1)  # keys that any query sees
    rows = b * d * (2 * h * t + 2 * kv * near)  # q, out; k, v
    # Forward two products; backward five, one of them the scores again. out, dout, dq as q; dk, dv as k.
    more = b * d * (2 * h * t + 2 * kv * s) if case["train"] else 0
    return {"bytes": size * (rows + more), "flops": (14 if case["train"] else 4) * d * pairs}
