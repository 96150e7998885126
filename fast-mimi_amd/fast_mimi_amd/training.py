"""Operators with gradients: LayerNorm, sliding-window attention, codebook embedding.

What a transformer over codec frames and the codebooks below it need to be
trained, on the HIP kernels of ``libfast_mimi_amd.so``:

* :func:`layer_norm`, :func:`window_attention` and :func:`code_embedding` are
  differentiable (``torch.autograd``, reverse mode, first order: dual tensors
  raise ``NotImplementedError``);
* ``*_forward`` / ``*_backward`` are the same without autograd, for a training
  loop that keeps its own tape, or that records its step in a hipGraph.

FP32, bfloat16 and float16 inputs; every sum, softmax state and statistic is
FP32 and each output is rounded once.  The same call gives the same bits.
Outputs and scratch memory are allocated by the call, on the current stream;
nothing synchronises.  Inputs must be on a ROCm GPU: there is no other backend.

In a hipGraph: torch gives a leaf's gradient on the stream on which the leaf
was first used, for as long as an autograd graph of it (or whoever else holds its
gradient accumulator) lives.  Where that is the default stream, which cannot be
captured, a captured backward pass of the same leaf ends the process: the
differentiable functions raise ``RuntimeError`` for a leaf that went through them
there first.  Warm up on a side stream, as ``torch.cuda.make_graphed_callables``
does, drop the eager graph, or capture the ``*_backward`` functions.
"""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native as nat
from . import ops

__all__ = [
    "code_embedding",
    "code_embedding_backward",
    "code_embedding_forward",
    "layer_norm",
    "layer_norm_backward",
    "layer_norm_forward",
    "window_attention",
    "window_attention_backward",
    "window_attention_forward",
]

_DEFAULT_STREAM = "fast_mimi_amd.default_stream"
_DTYPES = {torch.float32: nat.DTYPE_F32, torch.bfloat16: nat.DTYPE_BF16, torch.float16: nat.DTYPE_F16}


# ------------------------------------------------------------------- checks
def _reverse_mode(*tensors) -> None:
    """Refuses tensors with a forward-mode tangent, which would be lost without a word."""
    if forward_ad._current_level < 0:
        return
    if any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("the training operators have no forward-mode derivative: an input has a tangent")


def _tensor(name: str, t, dtypes=tuple(_DTYPES)) -> torch.Tensor:
    """``t`` as the kernels read it (no graph, no lazy negation), or TypeError."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d).replace('torch.', '') for d in dtypes)}, got {t.dtype}")
    _reverse_mode(t)
    if t.requires_grad:
        t = t.detach()
    return t.resolve_neg() if t.is_neg() else t


def _on_gpu(**tensors) -> torch.device:
    """The one GPU that all of the tensors (those that are given) are on."""
    device = None
    for name, t in tensors.items():
        if t is None:
            continue
        if t.device != device:
            if t.device.type != "cuda":
                raise ValueError(f"{name} must be on a ROCm GPU, got {t.device}")
            if device is not None:
                raise ValueError(f"{name} is on {t.device}, the other inputs on {device}")
            device = t.device
    return device


def _run(device: torch.device, entry: str, *args) -> None:
    """The entry point, with its tensors' device as the current one."""
    if device.index == torch.cuda.current_device():
        ops.call(entry, *args)
    else:
        with torch.cuda.device(device):
            ops.call(entry, *args)


def _scratch(like: torch.Tensor, entry: str, *args) -> tuple[torch.Tensor | None, int]:
    """Workspace for a call: what its size query asks for."""
    size = getattr(nat.library(), entry)(*args)
    return (like.new_empty((size + 3) // 4, dtype=torch.float32) if size else None), size


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``t`` as rows of its last dimension at one pitch (a copy where its
    strides allow none), and the pitch."""
    c = t.shape[-1]
    if t.numel() == 0 or t.is_contiguous():
        return t, c
    if t.stride(-1) == 1 or c == 1:
        # Leading dimensions that collapse into one.
        pitch, expect = None, None
        for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if size == 1:
                continue
            if pitch is None:
                pitch, expect = stride, stride * size
            elif stride != expect:
                pitch = None
                break
            else:
                expect *= size
        else:
            if pitch is None or pitch >= c:
                return t, c if pitch is None else pitch
    return t.contiguous(), c


def _accumulators(inputs):
    """The gradient accumulators of the leaves among ``inputs``: each lives as
    long as an autograd graph that uses its leaf."""
    for t in inputs:
        if t is not None and t.requires_grad and t.grad_fn is None:
            yield t.view_as(t).grad_fn.next_functions[0][0]


def _apply(function, inputs, *args):
    """``function.apply(*args)``, refused under stream capture for a leaf of
    ``inputs`` whose gradient would come on the default stream (see the module's
    text).  An accumulator keeps its stream, so the first use decides."""
    _reverse_mode(*inputs)  # a Function's forward does not see tangents
    capturing = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
    if capturing and any(node.metadata.get(_DEFAULT_STREAM) for node in _accumulators(inputs)):
        raise RuntimeError("a captured graph cannot use a leaf of an eager autograd graph that was made on the default stream "
                           "and is still alive: drop the eager graph (and what else holds the leaf's gradient accumulator), "
                           "make it on another stream, or capture the *_forward and *_backward functions")
    out = function.apply(*args)
    default = torch._C._cuda_getCurrentRawStream(out.device.index) == 0
    for node in _accumulators(inputs):
        node.metadata.setdefault(_DEFAULT_STREAM, default)
    return out


def _differentiable(*inputs) -> bool:
    return torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in inputs)


# ---------------------------------------------------------------- LayerNorm
def _norm_weights(x, weight, bias):
    given = [(n, t) for n, t in (("weight", weight), ("bias", bias)) if t is not None]
    out = []
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            t = _tensor(name, t, (x.dtype,) if x.dtype == torch.float32 else (x.dtype, torch.float32))
            if t.shape != x.shape[-1:]:
                raise ValueError(f"{name} must have shape {tuple(x.shape[-1:])}, got {tuple(t.shape)}")
            t = t.contiguous()
        out.append(t)
    if len(given) == 2 and out[0].dtype != out[1].dtype:
        raise TypeError(f"weight is {out[0].dtype}, bias {out[1].dtype}: they must have one type")
    wtype = next((t.dtype for t in out if t is not None), x.dtype)
    return out[0], out[1], wtype


def _norm_input(x, weight, bias):
    x = _tensor("x", x)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"x must have a last dimension to normalise, got shape {tuple(x.shape)}")
    weight, bias, wtype = _norm_weights(x, weight, bias)
    return x, weight, bias, wtype


def layer_norm_forward(x, weight=None, bias=None, eps: float = 1e-5):
    """``(y, mean, rstd)`` of LayerNorm over the last dimension of ``x``.

    ``weight`` and ``bias`` (each optional) have ``x``'s type or FP32; ``mean``
    and ``rstd`` are FP32, one per row, for :func:`layer_norm_backward`.
    """
    x, weight, bias, wtype = _norm_input(x, weight, bias)
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    device = _on_gpu(x=x, weight=weight, bias=bias)
    x, pitch = _rows(x)
    shape = x.shape
    y = x.new_empty(shape)
    mean = x.new_empty(shape[:-1], dtype=torch.float32)
    rstd = torch.empty_like(mean)
    rows = mean.numel()
    if rows:
        _run(device, "fm_layer_norm_forward", x, pitch, weight, bias, rows, shape[-1], float(eps), _DTYPES[x.dtype],
             _DTYPES[wtype], y, mean, rstd)
    return y, mean, rstd


def layer_norm_backward(grad, x, mean, rstd, weight=None, bias=None):
    """``(dx, dweight, dbias)`` for the gradient ``grad`` of the output of
    :func:`layer_norm_forward`; ``None`` for a weight or bias that was not given."""
    x, weight, bias, wtype = _norm_input(x, weight, bias)
    grad, mean, rstd = _tensor("grad", grad, (x.dtype,)), _tensor("mean", mean, (torch.float32,)), \
        _tensor("rstd", rstd, (torch.float32,))
    if grad.shape != x.shape:
        raise ValueError(f"grad must have x's shape {tuple(x.shape)}, got {tuple(grad.shape)}")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.shape != x.shape[:-1] or not t.is_contiguous():
            raise ValueError(f"{name} must be what layer_norm_forward returned for x")
    device = _on_gpu(x=x, grad=grad, mean=mean, rstd=rstd, weight=weight, bias=bias)
    (x, ld_x), (grad, ld_dy) = _rows(x), _rows(grad)
    dx = x.new_empty(x.shape)
    dw = None if weight is None else torch.empty_like(weight)
    db = None if bias is None else torch.empty_like(bias)
    rows, c = mean.numel(), x.shape[-1]
    ws, size = (None, 0) if dw is None and db is None else _scratch(x, "fm_layer_norm_backward_workspace_bytes", rows, c)
    _run(device, "fm_layer_norm_backward", grad, ld_dy, x, ld_x, weight, mean, rstd, rows, c, _DTYPES[x.dtype],
         _DTYPES[wtype], dx, dw, db, ws, size)
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        dx, dw, db = layer_norm_backward(grad, x, mean, rstd, weight, bias)
        return tuple(g if need else None for g, need in zip((dx, dw, db, None), ctx.needs_input_grad))


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """LayerNorm over the last dimension of ``x``, differentiable (see
    :func:`layer_norm_forward` for the types)."""
    if not _differentiable(x, weight, bias):
        return layer_norm_forward(x, weight, bias, eps)[0]
    return _apply(_LayerNorm, (x, weight, bias), x, weight, bias, eps)


# ---------------------------------------------------------------- attention
def _attention_input(q, k, v, window, scale, lengths):
    q = _tensor("q", q)
    k, v = _tensor("k", k, (q.dtype,)), _tensor("v", v, (q.dtype,))
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4:
            raise ValueError(f"{name} must be [batch, positions, heads, head_dim], got shape {tuple(t.shape)}")
    b, t, h, d = q.shape
    s, kv = k.shape[1], k.shape[2]
    if k.shape != (b, s, kv, d) or v.shape != k.shape:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    if t > s:
        raise ValueError(f"{t} queries over {s} keys: the queries are the last positions of the keys")
    if h == 0 or kv == 0 or h % kv:
        raise ValueError(f"{h} query heads are not a multiple of {kv} key heads")
    unit = 4 if q.dtype == torch.float32 else 8
    if not 0 < d <= 128 or d % unit:
        raise ValueError(f"head_dim must be a multiple of {unit} up to 128 for {q.dtype}, got {d}")
    if window is None:
        window = max(s, 1)
    if not isinstance(window, int) or isinstance(window, bool) or window <= 0:
        raise ValueError(f"window must be a positive integer or None, got {window!r}")
    window = min(window, max(s, 1))
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    if lengths is not None:
        lengths = _tensor("lengths", lengths, (torch.int32,))
        if lengths.shape != (b,):
            raise ValueError(f"lengths must have shape ({b},), got {tuple(lengths.shape)}")
        lengths = lengths.contiguous()
    return q, k, v, window, scale, lengths


def _heads(t: torch.Tensor, group: int = 1) -> tuple[torch.Tensor, int, int, int]:
    """``t`` [B, N, H, D] with its batch, position and head strides as the
    kernels take them: 16-byte rows within 32-bit reach, else a copy."""
    size = t.element_size()
    unit = 16 // size
    b, n, h, d = t.shape
    sb, sn, sh, sd = t.stride()
    # The stride of a single item does not matter, whatever it says (also of a copy).
    sb, sn, sh = sb if b > 1 else 0, sn if n > 1 else 0, sh if h > 1 else 0
    reach = 0x7fffffff // size
    if (sd != 1 and d > 1) or (sb | sn | sh) % unit or t.data_ptr() % 16 or sn > reach // 256 or sh > reach // 2 // group:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        sb, sn, sh = n * h * d if b > 1 else 0, h * d if n > 1 else 0, d if h > 1 else 0
    return t, sb, sn, sh


def window_attention_forward(q, k, v, window: int | None = None, scale: float | None = None, lengths=None):
    """``(out, lse)`` of causal sliding-window attention.

    ``q`` is ``[batch, queries, heads, head_dim]``, ``k`` and ``v`` are
    ``[batch, keys, kv_heads, head_dim]`` (any strides; slices of a packed
    projection are read in place).  The queries are the last positions of the
    keys: query ``t`` is at ``p = keys - queries + t`` and sees key ``j`` iff
    ``p - window < j <= p`` (``window=None``: every earlier key).  ``lengths``
    (int32 ``[batch]``): positions from ``lengths[b]`` on are padding; it is
    never read, its rows of ``out`` are zeros.  ``scale`` defaults to
    ``head_dim ** -0.5``.  ``lse`` (FP32 ``[batch, queries, heads]``, base 2) is
    for :func:`window_attention_backward`.

    An infinity or NaN may reach other rows near it; what padding holds
    reaches nothing.  At most 2097120 keys, and queries times
    heads per key head.
    """
    q, k, v, window, scale, lengths = _attention_input(q, k, v, window, scale, lengths)
    device = _on_gpu(q=q, k=k, v=v, lengths=lengths)
    b, t, h, d = q.shape
    s, kv = k.shape[1], k.shape[2]
    out = q.new_empty((b, t, h, d))
    lse = q.new_empty((b, t, h), dtype=torch.float32)
    if b and t:
        ws, size = _scratch(q, "fm_attention_forward_workspace_bytes", b, t, s, h, kv, d, window)
        _run(device, "fm_attention_forward", *_heads(q, h // kv), *_heads(k), *_heads(v), lengths, b, t, s, h, kv, d, window,
             scale, _DTYPES[out.dtype], out, lse, ws, size)
    return out, lse


def window_attention_backward(grad, q, k, v, out, lse, window: int | None = None, scale: float | None = None, lengths=None):
    """``(dq, dk, dv)`` for the gradient ``grad`` of the output of
    :func:`window_attention_forward` (``out``, ``lse``: what it returned).
    """
    q, k, v, window, scale, lengths = _attention_input(q, k, v, window, scale, lengths)
    grad, out, lse = _tensor("grad", grad, (q.dtype,)), _tensor("out", out, (q.dtype,)), _tensor("lse", lse, (torch.float32,))
    b, t, h, d = q.shape
    s, kv = k.shape[1], k.shape[2]
    if grad.shape != q.shape:
        raise ValueError(f"grad must have q's shape {tuple(q.shape)}, got {tuple(grad.shape)}")
    if out.shape != q.shape or lse.shape != (b, t, h) or not lse.is_contiguous():
        raise ValueError("out and lse must be what window_attention_forward returned for q, k and v")
    device = _on_gpu(q=q, k=k, v=v, grad=grad, out=out, lse=lse, lengths=lengths)
    dq, dk, dv = q.new_empty((b, t, h, d)), q.new_empty((b, s, kv, d)), q.new_empty((b, s, kv, d))
    if b and s:
        if t == 0:
            return dq, dk.zero_(), dv.zero_()
        out = _heads(out.contiguous())[0]
        stats = lse.new_empty((2, b, t, h))
        _run(device, "fm_attention_backward", *_heads(grad, h // kv), *_heads(q, h // kv), *_heads(k), *_heads(v), out, lse,
             lengths, b, t, s, h, kv, d, window, scale, _DTYPES[q.dtype], dq, dk, dv, stats)
    return dq, dk, dv


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, scale, lengths):
        out, lse = window_attention_forward(q, k, v, window, scale, lengths)
        ctx.save_for_backward(q, k, v, out, lse, lengths)
        ctx.how = window, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, out, lse, lengths = ctx.saved_tensors
        grads = window_attention_backward(grad, q, k, v, out, lse, *ctx.how, lengths)
        return tuple(g if need else None for g, need in zip((*grads, None, None, None), ctx.needs_input_grad))


def window_attention(q, k, v, window: int | None = None, scale: float | None = None, lengths=None):
    """Causal sliding-window attention, differentiable in ``q``, ``k`` and ``v``
    (see :func:`window_attention_forward` for the layouts and the mask)."""
    if not _differentiable(q, k, v):
        return window_attention_forward(q, k, v, window, scale, lengths)[0]
    return _apply(_WindowAttention, (q, k, v), q, k, v, window, scale, lengths)


# ------------------------------------------------------- codebook embedding
def _embedding_input(codes, table, scale):
    table = _tensor("table", table)
    codes = _tensor("codes", codes, (torch.int64,))
    if codes.dim() != 3:
        raise ValueError(f"codes must be [batch, codebooks, frames], got shape {tuple(codes.shape)}")
    if table.dim() != 3 or 0 in table.shape:
        raise ValueError(f"table must be [codebooks, entries, dim], got shape {tuple(table.shape)}")
    if codes.shape[1] != table.shape[0]:
        raise ValueError(f"codes have {codes.shape[1]} codebooks, table {table.shape[0]}")
    if table.shape[1] > 32768:
        raise ValueError(f"a codebook may have at most 32768 entries, got {table.shape[1]}")
    scale = float(scale)
    if math.isnan(scale):
        raise ValueError("scale is not a number")
    if codes.numel() and codes.stride(2) != 1 and codes.shape[2] > 1:
        codes = codes.contiguous()
    return codes, table, scale


def code_embedding_forward(codes, table, scale: float = 1.0):
    """``scale * sum_q table[q, codes[:, q]]``: ``[batch, frames, dim]`` of ``table``'s type.

    ``codes`` is int64 ``[batch, codebooks, frames]``, ``table``
    ``[codebooks, entries, dim]`` (at most 32768 entries; 2097120 frames in
    all).  Code -1 is absent
    and adds nothing (padding, delayed codebooks); any other code outside the
    table makes its frame NaN, as ``rvq_decode`` does.  The split quantizer's
    two sums are two calls, on ``codes[:, :n]`` / ``table[:n]`` and the rest.
    """
    codes, table, scale = _embedding_input(codes, table, scale)
    device = _on_gpu(codes=codes, table=table)
    (b, books, frames), (_, entries, dim) = codes.shape, table.shape
    out = table.new_empty((b, frames, dim))
    if b and frames:
        _run(device, "fm_code_embedding", codes, codes.stride(0), codes.stride(1), b, books, frames, table.contiguous(),
             entries, dim, scale, _DTYPES[table.dtype], out)
    return out


def code_embedding_backward(grad, codes, table, scale: float = 1.0):
    """The gradient of ``table`` for the gradient ``grad`` ``[batch, frames,
    dim]`` of :func:`code_embedding_forward`'s output: each entry's rows, summed
    in their order; zeros for entries that no frame has.  Of ``table`` only the
    shape, type and device count."""
    codes, table, scale = _embedding_input(codes, table, scale)
    grad = _tensor("grad", grad, (table.dtype,))
    (b, books, frames), (_, entries, dim) = codes.shape, table.shape
    if grad.shape != (b, frames, dim):
        raise ValueError(f"grad must have shape {(b, frames, dim)}, got {tuple(grad.shape)}")
    device = _on_gpu(codes=codes, table=table, grad=grad)
    grad, pitch = _rows(grad)
    dtable = table.new_empty(table.shape)
    ws, size = _scratch(grad, "fm_code_embedding_backward_workspace_bytes", b, books, frames, entries, dim)
    _run(device, "fm_code_embedding_backward", grad, pitch, codes, codes.stride(0), codes.stride(1), b, books, frames, entries,
         dim, scale, _DTYPES[table.dtype], dtable, ws, size)
    return dtable


class _CodeEmbedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, codes, scale):
        ctx.save_for_backward(codes)
        # Of the table only the shape matters: it may change before the backward pass.
        ctx.how = table.detach(), scale
        return code_embedding_forward(codes, table, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return code_embedding_backward(grad, *ctx.saved_tensors, *ctx.how), None, None


def code_embedding(codes, table, scale: float = 1.0):
    """The scaled sum of each frame's codebook entries, differentiable in
    ``table`` (see :func:`code_embedding_forward`)."""
    if not _differentiable(table):
        return code_embedding_forward(codes, table, scale)
    return _apply(_CodeEmbedding, (table,), table, codes, scale)
