"""RMS norm, rotary positions, cross attention and 8-bit products from their definitions in 64
bits, with elementwise bounds on what FP32 sums and roundings to the outputs' types may add
(see training_ref, whose ``H``, ``half`` and ``step0`` these are)."""

from __future__ import annotations

import torch

from training_ref import H, half, step0

BLOCK = 128


# ----------------------------------------------------------------- RMS norm
def rms(x, residual, weight, grad, grad_h, eps):
    """(values, bounds): y, h, dx, dresidual, dweight of rows [N, C] in float64."""
    t = x.dtype
    st = t if residual is None else residual.dtype
    wt = t if weight is None else weight.dtype
    x, grad = x.double().cpu(), grad.double().cpu()
    n, c = x.shape
    r = torch.zeros_like(x) if residual is None else residual.double().cpu()
    w = torch.ones(c, dtype=torch.float64) if weight is None else weight.double().cpu()
    gh = torch.zeros_like(x) if grad_h is None else grad_h.double().cpu()
    h = x + r
    rstd = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    hh, g = h * rstd, grad * w
    m = (g * hh).mean(1, keepdim=True)
    inner = g - hh * m
    y, dh, dw = hh * w, gh + rstd * inner, (grad * hh).sum(0)
    # A row's sum runs over at most C / 16 values a lane, then at most 8 joins; each value is off by
    # two roundings (the sum x + residual, and h's own where the backward pass gets that) before its square.
    k = c / 16 + 10
    r_rstd = (k + 4) * H / 2 + 2 * H + 3 * H
    e_hh = hh.abs() * (r_rstd + 3 * H)
    e_y = e_hh * w.abs() + 2 * H * y.abs() + half(t) * y.abs() + step0(t)
    e_h = H * h.abs() + half(st) * h.abs() + step0(st)
    e_m = (k + 3) * H * (g * hh).abs().mean(1, keepdim=True) + (g.abs() * e_hh).mean(1, keepdim=True)
    e_dh = rstd * (e_m * hh.abs() + e_hh * m.abs() + 4 * H * (g.abs() + (hh * m).abs())) + rstd * inner.abs() * (r_rstd + 2 * H) \
        + 2 * H * (dh.abs() + gh.abs())
    e_dw = (n + 2) * H * (grad * hh).abs().sum(0) + (grad.abs() * e_hh).sum(0) + half(wt) * dw.abs() + step0(wt)
    val = {"y": y, "h": h, "dx": dh, "dresidual": dh, "dweight": dw}
    err = {"y": e_y, "h": e_h, "dx": e_dh + half(t) * dh.abs() + step0(t),
           "dresidual": e_dh + half(st) * dh.abs() + step0(st), "dweight": e_dw}
    return val, err


# --------------------------------------------------------- rotary positions
def rotary(x, frequencies, positions, interleaved, scale, inverse=False):
    """(value, bound) of x [B, T, H, D] turned by positions [B, T]."""
    t = x.dtype
    x = x.double().cpu()
    pairs = frequencies.numel()
    # Angles beyond 2^53 roundings: whole turns are taken off in Python's integers.
    angle = torch.empty((*positions.shape, pairs), dtype=torch.float64)
    from fractions import Fraction

    turn = Fraction(6283185307179586476925286766559005768394338798750211641949889, 10 ** 60)
    for i, p in enumerate(positions.reshape(-1).tolist()):
        for j, f in enumerate(frequencies.tolist()):
            a = Fraction(f) * p
            angle.view(-1, pairs)[i, j] = float(a - turn * round(a / turn))
    cos, sin = (torch.cos(angle) * scale)[:, :, None], (torch.sin(angle) * scale * (-1 if inverse else 1))[:, :, None]
    out, size = x.clone(), torch.zeros_like(x)
    a, b = (x[..., 0: 2 * pairs: 2], x[..., 1: 2 * pairs: 2]) if interleaved else (x[..., :pairs], x[..., pairs: 2 * pairs])
    at = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    out[..., at[0]], out[..., at[1]] = a * cos - b * sin, b * cos + a * sin
    for s in at:
        size[..., s] = (a.abs() + b.abs()) * abs(scale)
    # Sine and cosine within 3.5 H each (the angle's rounding and the polynomials' six), a product and a sum.
    turned = size > 0
    return out, 6 * H * size + torch.where(turned, half(t) * (out.abs() + 6 * H * size) + step0(t), 0.0)


# ---------------------------------------------------------- cross attention
def cross(q, k, v, grad, scale, key_lengths, query_lengths, pieces=1):
    """(values, bounds): out, dq, dk, dv in float64; padding is not read.  The bounds are those of
    training_ref.attention, whose kernels' arithmetic this is."""
    t = q.dtype
    b, tq, h, d = q.shape
    s, kv = k.shape[1], k.shape[2]
    n = h // kv
    u = half(t)
    up, eta = (0.0, 2.0 ** -126) if t == torch.float32 else (u, max(step0(t), 2.0 ** -126))
    du = u
    if pieces == 2:
        up, du = up * up, 0.0
    val = {m: torch.zeros(x.shape, dtype=torch.float64) for m, x in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    err = {m: torch.zeros_like(x) for m, x in val.items()}
    q, k, v, grad = (x.double().cpu() for x in (q, k, v, grad))
    for i in range(b):
        rows = tq if query_lengths is None else min(max(int(query_lengths[i]), 0), tq)
        keys = s if key_lengths is None else min(max(int(key_lengths[i]), 0), s)
        if rows == 0 or keys == 0:
            continue
        for a in range(h):
            c = a // n
            Q, K, V, G = q[i, :rows, a], k[i, :keys, c], v[i, :keys, c], grad[i, :rows, a]
            S = (Q @ K.T) * scale
            lse = S.logsumexp(1, keepdim=True)
            P = torch.exp(S - lse)
            O = P @ V
            es = (d + 4) * H * (Q.abs() @ K.abs().T) * scale + 2 * H * lse.abs()
            ep = P * (es + es.amax(1, keepdim=True) + (keys + 12) * H)
            eo = (ep + (up + (keys + 4) * H) * P + eta) @ V.abs()
            DP = G @ V.T
            D = (G * O).sum(1, keepdim=True)
            DS = P * (DP - D)
            edp = (d + 2) * H * (G.abs() @ V.abs().T)
            eD = (G.abs() * (du * O.abs() + eo + step0(t) + (d + 2) * H * O.abs())).sum(1, keepdim=True)
            # A probability below 2^-126 is zero (eta): dS = P (dP - D) loses up to eta |dP - D| with it.  (Scores of
            # 739 under a largest of 826 have P = 1.1e-38 and dP - D = 17.)  Its own rounding near zero is the other eta.
            eds = ep * (DP - D).abs() + P * (edp + eD + 2 * H * (DP.abs() + D.abs())) + (up + 2 * H) * DS.abs() \
                + eta * ((DP - D).abs() + 1)
            val["out"][i, :rows, a] = O
            err["out"][i, :rows, a] = eo + u * O.abs() + step0(t)
            val["dq"][i, :rows, a] = DS @ K * scale
            err["dq"][i, :rows, a] = (eds + (keys + 3) * H * DS.abs()) @ K.abs() * scale
            val["dk"][i, :keys, c] += DS.T @ Q * scale
            err["dk"][i, :keys, c] += (eds + (n * rows + 3) * H * DS.abs()).T @ Q.abs() * scale
            val["dv"][i, :keys, c] += P.T @ G
            err["dv"][i, :keys, c] += (ep + (up + (n * rows + 3) * H) * P + eta).T @ G.abs()
    for m in ("dq", "dk", "dv"):
        err[m] += torch.where(err[m] > 0, u * (val[m].abs() + err[m]) + step0(t), 0.0)
    return val, err


# -------------------------------------------------------------------- 8 bits
def exponents(most):
    """The least e >= -127 with most <= 448 * 2^e."""
    m, x = torch.frexp(most.double())
    return torch.where(most == 0, -127, x - 9 + (m > 0.875).int()).clamp(min=-127)


def in_8_bits(x, rows):
    """(values, scale bytes) of float64 x [R, C], `rows` rows and 128 channels to a scale, ties to even."""
    r, c = x.shape
    pad = torch.nn.functional.pad(x, (0, -c % BLOCK, 0, -r % rows))
    blocks = pad.reshape(pad.shape[0] // rows, rows, pad.shape[1] // BLOCK, BLOCK)
    e = exponents(blocks.abs().amax((1, 3)))
    v = blocks * torch.exp2(-e.double())[:, None, :, None]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).reshape(pad.shape)[:r, :c], e + 127


def stand_for(values, scales, rows):
    """What 8-bit values [R, C] and their scales stand for, in float64."""
    full = torch.exp2(scales.cpu().view(torch.uint8).double() - 127).repeat_interleave(rows, 0).repeat_interleave(BLOCK, 1)
    return values.cpu().double() * full[: values.shape[0], : values.shape[1]]


def product(x, w, dtype):
    """(value, bound) of x [M, K] @ w [N, K]^T, both what 8-bit values stand for.

    The 8-bit matrix instructions line up eight products by their largest and drop what lies
    2^-13 below it, each time they add eight to an FP32 sum; FP32 results are summed from
    exact products."""
    k = x.shape[1]
    y = x @ w.T
    size = x.abs() @ w.abs().T
    bound = (k + 2) * H * size
    if dtype != torch.float32:
        groups = torch.nn.functional.pad(x.abs(), (0, -k % 8)).reshape(x.shape[0], -1, 8)
        others = torch.nn.functional.pad(w.abs(), (0, -k % 8)).reshape(w.shape[0], -1, 8)
        for g in range(groups.shape[1]):
            bound += 8 * 2.0 ** -13 * (groups[:, g, None] * others[None, :, g]).amax(2)
    return y, bound + half(dtype) * y.abs() + step0(dtype)
