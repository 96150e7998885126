"""The training operators from their definitions in 64 bits, with elementwise
bounds on what FP32 sums and roundings to the outputs' types may add.

``H`` is the half step of FP32, ``half(t)`` that of a type: every rounding is
off by at most that much of the value.  A sum of n products held in FP32 is off
by at most n H times the sum of their magnitudes, whatever its order.
"""

from __future__ import annotations

import torch

H = 2.0 ** -24
# First-order bounds leave out products of errors (below 1e-3 of them here).
SECOND_ORDER = 1.01


def half(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def step0(dtype) -> float:
    """Half the smallest step of a type: what rounding loses near zero."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def assert_within(name, got, want, bound):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    off = (got - want).abs()
    bound = bound.detach().double().cpu().expand_as(off)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    worst = (off - SECOND_ORDER * bound).max().item() if off.numel() else 0.0
    at = (off / (bound + 1e-300)).max().item() if off.numel() else 0.0
    assert worst <= 0, f"{name}: {at:.3g} times its bound"


# ---------------------------------------------------------------- LayerNorm
def norm(x, grad, weight, bias, eps):
    """(values, bounds): y, dx, dw, db of rows x [N, C] in float64."""
    t, wt = x.dtype, (weight if weight is not None else bias if bias is not None else x).dtype
    x, grad = x.double().cpu(), grad.double().cpu()
    n, c = x.shape
    w = torch.ones(c, dtype=torch.float64) if weight is None else weight.double().cpu()
    b = torch.zeros(c, dtype=torch.float64) if bias is None else bias.double().cpu()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    xh = d * rstd
    g = grad * w
    m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    y, dx = xh * w + b, rstd * (g - m1 - xh * m2)
    dw, db = (grad * xh).sum(0), grad.sum(0)

    # A row's sums run over at most C / 16 values a lane, then at most 8 joins.
    k = c / 16 + 10
    e_mean = k * H * x.abs().mean(1, keepdim=True)
    e_d = e_mean + H * d.abs()
    # rstd: the variance's relative error is that of its terms and its sum, halved by the root.
    var = (d * d).mean(1, keepdim=True) + eps
    r_rstd = ((d.abs() * e_d).mean(1, keepdim=True) + (k + 2) * H * var) / var + 3 * H
    e_xh = rstd * e_d + xh.abs() * (r_rstd + H)
    u, uw = half(t), half(wt)
    e_y = e_xh * w.abs() + 2 * H * ((xh * w).abs() + b.abs()) + u * y.abs() + step0(t)
    e_m1 = (k + 1) * H * g.abs().mean(1, keepdim=True)
    e_m2 = (k + 3) * H * (g * xh).abs().mean(1, keepdim=True) + (g.abs() * e_xh).mean(1, keepdim=True)
    inner = (g - m1 - xh * m2).abs()
    e_dx = rstd * (e_m1 + e_m2 * xh.abs() + e_xh * m2.abs() + 3 * H * (g.abs() + m1.abs() + (xh * m2).abs())) \
        + rstd * inner * (r_rstd + 2 * H)
    e_dx = e_dx + u * dx.abs() + step0(t)
    # Column sums: any order of n rows.
    e_dw = (n + 2) * H * (grad * xh).abs().sum(0) + (grad.abs() * e_xh).sum(0) + uw * dw.abs() + step0(wt)
    e_db = (n + 2) * H * grad.abs().sum(0) + uw * db.abs() + step0(wt)
    return {"y": y, "dx": dx, "dw": dw, "db": db}, {"y": e_y, "dx": e_dx, "dw": e_dw, "db": e_db}


# ---------------------------------------------------------------- attention
def visible(queries, keys, window, length):
    p = torch.arange(keys - queries, keys)[:, None]
    j = torch.arange(keys)[None]
    ok = (j <= p) & (p < length)
    return ok if window is None else ok & (j > p - window)


def attention(q, k, v, grad, window, scale, lengths, pieces=1):
    """(values, bounds): out, dq, dk, dv in float64; padding is not read.

    pieces=2: the gradients' bounds where 16-bit inputs keep P and dS in two
    pieces (of relative error u^2 together) and delta is the sum over P dP.
    """
    t = q.dtype
    b, tq, h, d = q.shape
    s, kv = k.shape[1], k.shape[2]
    n = h // kv
    u = half(t)
    # FP32 inputs keep their probabilities in FP32; the hardware's exponential
    # gives zero for results below FP32's smallest normal number, 2^-126.
    up, eta = (0.0, 2.0 ** -126) if t == torch.float32 else (u, max(step0(t), 2.0 ** -126))
    du = u
    if pieces == 2:
        up, du = up * up, 0.0
    val = {m: torch.zeros(x.shape, dtype=torch.float64) for m, x in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    err = {m: torch.zeros_like(x) for m, x in val.items()}
    q, k, v, grad = (x.double().cpu() for x in (q, k, v, grad))
    for i in range(b):
        length = s if lengths is None else min(max(int(lengths[i]), 0), s)
        see = visible(tq, s, window, length)
        live = see.any(1)
        for a in range(h):
            c = a // n
            Q, K, V, G = q[i, :, a], k[i, :, c].clone(), v[i, :, c].clone(), grad[i, :, a].clone()
            K[length:], V[length:] = 0, 0
            Q = torch.where(live[:, None], Q, 0.0)
            G = torch.where(live[:, None], G, 0.0)
            S = (Q @ K.T) * scale
            P = torch.where(see, torch.exp(S - torch.where(see, S, -torch.inf).amax(1, keepdim=True).nan_to_num(neginf=0.0)), 0.0)
            L = P.sum(1, keepdim=True)
            lse = torch.where(see, S, -torch.inf).logsumexp(1, keepdim=True).nan_to_num(neginf=0.0)
            P = P / torch.where(L == 0, 1.0, L)
            O = P @ V
            # Scores: d products, the scale and the exponent's subtraction.
            es = ((d + 4) * H * (Q.abs() @ K.abs().T) * scale + 2 * H * lse.abs()) * see
            ep = P * (es + es.amax(1, keepdim=True) + (s + 12) * H)
            eo = (ep + (up + (s + 4) * H) * P + eta * see) @ V.abs()
            DP = G @ V.T
            D = (G * O).sum(1, keepdim=True)
            DS = P * (DP - D)
            edp = (d + 2) * H * (G.abs() @ V.abs().T)
            eD = (G.abs() * (du * O.abs() + eo + step0(t) + (d + 2) * H * O.abs())).sum(1, keepdim=True)
            eds = ep * (DP - D).abs() + P * (edp + eD + 2 * H * (DP.abs() + D.abs())) + (up + 2 * H) * DS.abs() + eta * see
            val["out"][i, :, a] = O
            err["out"][i, :, a] = eo + u * O.abs() + step0(t)
            val["dq"][i, :, a] = DS @ K * scale
            err["dq"][i, :, a] = (eds + (s + 3) * H * DS.abs()) @ K.abs() * scale
            val["dk"][i, :, c] += DS.T @ Q * scale
            err["dk"][i, :, c] += (eds + (n * tq + 3) * H * DS.abs()).T @ Q.abs() * scale
            val["dv"][i, :, c] += P.T @ G
            err["dv"][i, :, c] += (ep + (up + (n * tq + 3) * H) * P + eta * see).T @ G.abs()
    for m in ("dq", "dk", "dv"):
        err[m] += u * (val[m].abs() + err[m]) + step0(t)
    return val, err


# ------------------------------------------------------- codebook embedding
def embedding(codes, table, grad, scale):
    """(values, bounds): out, dtable in float64; codes below 0 are absent."""
    t = table.dtype
    codes, table, grad = codes.cpu(), table.double().cpu(), grad.double().cpu()
    b, books, frames = codes.shape
    out = torch.zeros(b, frames, table.shape[2], dtype=torch.float64)
    size, dtable, gsize = torch.zeros_like(out), torch.zeros_like(table), torch.zeros_like(table)
    count = torch.zeros(table.shape[:2], dtype=torch.float64)
    for j in range(books):
        at = codes[:, j] >= 0
        picked = table[j][codes[:, j][at]]
        out[at] += picked
        size[at] += picked.abs()
        dtable[j].index_add_(0, codes[:, j][at], grad[at])
        gsize[j].index_add_(0, codes[:, j][at], grad[at].abs())
        count[j].index_add_(0, codes[:, j][at], torch.ones(int(at.sum()), dtype=torch.float64))
    u, a = half(t), abs(scale)
    e_out = (books + 2) * H * size * a + u * out.abs() * a + step0(t)
    e_table = (count[..., None] + 2) * H * gsize * a + u * dtable.abs() * a + step0(t)
    return {"out": out * scale, "dtable": dtable * scale}, {"out": e_out, "dtable": e_table}
