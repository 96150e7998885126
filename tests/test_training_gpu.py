"""The training operators (``fast_mimi_amd.training``) on the GPU against their
definitions in 64 bits (``training_ref``), elementwise, within what FP32 sums
and the roundings to the outputs' types may add."""

from __future__ import annotations

import math

import pytest
import torch

import training_ref as ref
from fast_mimi_amd import training as tr

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def check(got: dict, want_bounds):
    want, bound = want_bounds
    for name, t in got.items():
        ref.assert_within(name, t, want[name], bound[name])


# ---------------------------------------------------------------- LayerNorm
def norm_case(rows, c, dtype, wtype, seed=0, weight=True, bias=True):
    g = gen(seed)
    x = (torch.randn(rows, c, generator=g) * (0.5 + torch.rand(rows, 1, generator=g)) + 0.4 * torch.randn(c, generator=g))
    w = (1 + 0.2 * torch.randn(c, generator=g)).to(wtype).to(DEV) if weight else None
    b = (0.2 * torch.randn(c, generator=g)).to(wtype).to(DEV) if bias else None
    return x.to(dtype).to(DEV), torch.randn(rows, c, generator=g).to(dtype).to(DEV), w, b


def norm_run(x, grad, w, b, eps=1e-5):
    y, mean, rstd = tr.layer_norm_forward(x, w, b, eps)
    dx, dw, db = tr.layer_norm_backward(grad, x, mean, rstd, w, b)
    return {n: t for n, t in (("y", y), ("dx", dx), ("dw", dw), ("db", db)) if t is not None}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,c", [(1, 1), (1, 512), (13, 512), (33, 8), (257, 64), (40, 100), (70, 513), (5, 2047), (67, 2048),
                                    (3, 2049), (9, 4096), (2, 8200), (1500, 256)])
def test_layer_norm(rows, c, dtype):
    x, grad, w, b = norm_case(rows, c, dtype, dtype)
    check(norm_run(x, grad, w, b), ref.norm(x, grad, w, b, 1e-5))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 8, 9, 32, 33, 1100])
@pytest.mark.parametrize("c", [511, 516, 1023, 1028, 2049, 2052, 4099, 4104, 8191, 8192, 8193, 8200])
def test_layer_norm_plans(rows, c, dtype):
    """Every number of lanes and vectors per row, at its edges, alone and in many blocks."""
    x, grad, w, b = norm_case(rows, c, dtype, torch.float32, rows)
    check(norm_run(x, grad, w, b), ref.norm(x, grad, w, b, 1e-5))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("weight,bias", [(True, True), (True, False), (False, True), (False, False)])
def test_layer_norm_fp32_weights(dtype, weight, bias):
    for c in (512, 77):
        x, grad, w, b = norm_case(50, c, dtype, torch.float32, 1, weight, bias)
        got = norm_run(x, grad, w, b)
        assert set(got) == {"y", "dx"} | ({"dw"} if weight else set()) | ({"db"} if bias else set())
        check(got, ref.norm(x, grad, w, b, 1e-5))


def test_layer_norm_offset_rows_keep_their_variance():
    """Rows around a large mean: the variance is that of the centred values."""
    x, grad, w, b = norm_case(20, 512, torch.float32, torch.float32, 2)
    x = x + 300.0
    check(norm_run(x, grad, w, b), ref.norm(x, grad, w, b, 1e-5))


def test_layer_norm_constant_rows():
    x, grad, w, b = norm_case(6, 512, torch.float32, torch.float32, 3)
    x[1], x[3] = 0.0, 2.0
    check(norm_run(x, grad, w, b), ref.norm(x, grad, w, b, 1e-5))


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_strided_inputs(dtype):
    """A column slice (aligned and not), a 3-D view, a transposed view, an expanded gradient."""
    g = gen(4)
    wide = torch.randn(30, 1100, generator=g).to(dtype).to(DEV)
    w, b = torch.randn(512, generator=g).to(dtype).to(DEV), torch.randn(512, generator=g).to(dtype).to(DEV)
    for x in (wide[:, 64:576], wide[:, 3:515], wide[::3, 8:520]):
        grad = wide[:x.shape[0], 500:1012]
        check(norm_run(x, grad, w, b), ref.norm(x, grad, w, b, 1e-5))
    cube = torch.randn(4, 512, 6, generator=g).to(dtype).to(DEV).transpose(1, 2)
    grad = torch.randn(1, 1, 512, generator=g).to(dtype).to(DEV).expand(4, 6, 512)
    got = norm_run(cube, grad, w, b)
    want = ref.norm(cube.reshape(24, 512), grad.reshape(24, 512), w, b, 1e-5)
    check({n: t.reshape(24, 512) if t.dim() == 3 else t for n, t in got.items()}, want)


def test_layer_norm_empty():
    w = torch.ones(512, device=DEV)
    y, mean, rstd = tr.layer_norm_forward(torch.empty(0, 512, device=DEV), w, w)
    assert y.shape == (0, 512) and mean.shape == (0,)
    dx, dw, db = tr.layer_norm_backward(y, y, mean, rstd, w, w)
    assert dx.shape == (0, 512) and not dw.any() and not db.any()


def test_layer_norm_nan_stays_in_its_row():
    x, grad, w, b = norm_case(9, 512, torch.float32, torch.float32, 5)
    clean = norm_run(x, grad, w, b)
    x[4, 7] = math.nan
    got = norm_run(x, grad, w, b)
    rest = [i for i in range(9) if i != 4]
    assert torch.equal(got["y"][rest], clean["y"][rest]) and torch.equal(got["dx"][rest], clean["dx"][rest])
    assert got["y"][4].isnan().all()


def test_layer_norm_many_elements():
    """More than 2^31 elements: the last rows are as a small call's."""
    rows, c = 4_200_003, 512
    x = torch.zeros(rows, c, dtype=torch.float16, device=DEV)
    tail, grad, w, b = norm_case(5, c, torch.float16, torch.float32, 6)
    x[-5:] = tail
    y, mean, rstd = tr.layer_norm_forward(x, w, b)
    assert torch.equal(y[-5:], tr.layer_norm_forward(tail, w, b)[0])
    g = torch.zeros_like(x)
    g[-5:] = grad
    got = dict(zip(("dx", "dw", "db"), tr.layer_norm_backward(g, x, mean, rstd, w, b)))
    got["dx"] = got["dx"][-5:]
    check(got, ref.norm(tail, grad, w, b, 1e-5))


def test_layer_norm_more_rows_than_a_grid_holds():
    rows, c = (1 << 24) + 9, 8
    tail, _, w, b = norm_case(7, c, torch.bfloat16, torch.float32, 7)
    x = torch.zeros(rows, c, dtype=torch.bfloat16, device=DEV)
    first = 1 << 23
    for at in (0, first - 7, first, rows - 7):
        x[at:at + 7] = tail
    got, want = tr.layer_norm_forward(x, w, b), tr.layer_norm_forward(tail, w, b)
    for at in (0, first - 7, first, rows - 7):
        assert all(torch.equal(t[at:at + 7], s) for t, s in zip(got, want)), at


# ---------------------------------------------------------------- attention
def attention_case(b, t, s, h, kv, d, dtype, seed=0, packed=False):
    g = gen(seed)
    if packed:
        assert t == s
        qkv = torch.randn(b, t, (h + 2 * kv) * d, generator=g).to(dtype).to(DEV)
        q = qkv[..., :h * d].view(b, t, h, d)
        k = qkv[..., h * d:(h + kv) * d].view(b, s, kv, d)
        v = qkv[..., (h + kv) * d:].view(b, s, kv, d)
    else:
        q, k, v = (torch.randn(n, generator=g).to(dtype).to(DEV) for n in ((b, t, h, d), (b, s, kv, d), (b, s, kv, d)))
    return q, k, v, torch.randn(b, t, h, d, generator=g).to(dtype).to(DEV)


def attention_run(q, k, v, grad, window, scale=None, lengths=None):
    out, lse = tr.window_attention_forward(q, k, v, window, scale, lengths)
    dq, dk, dv = tr.window_attention_backward(grad, q, k, v, out, lse, window, scale, lengths)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


SHAPES = [
    # b, t, s, heads, kv heads, dim, window
    (1, 1, 1, 1, 1, 64, None),
    (2, 13, 13, 8, 8, 64, 250),
    (1, 33, 33, 2, 1, 64, 1),
    (2, 65, 65, 4, 2, 32, 7),
    (1, 129, 129, 3, 3, 64, 32),
    (1, 250, 250, 2, 2, 64, 250),
    (1, 300, 300, 2, 1, 128, 100),
    (1, 97, 97, 6, 2, 72, None),
    (2, 31, 31, 2, 2, 8, 5),
    (1, 1, 700, 8, 2, 64, None),
    (2, 1, 40, 4, 4, 64, 16),
    (1, 5, 333, 6, 2, 128, None),
    (1, 100, 231, 2, 2, 64, 50),
    (1, 70, 500, 1, 1, 64, None),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(shape, dtype):
    *sizes, window = shape
    q, k, v, grad = attention_case(*sizes, dtype)
    check(attention_run(q, k, v, grad, window), ref.attention(q, k, v, grad, window, sizes[-1] ** -0.5, None))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,t,h,kv,d,window", [(40, 160, 8, 8, 64, 90), (20, 140, 16, 8, 128, None), (24, 140, 16, 16, 64, 60),
                                               (50, 70, 32, 16, 128, None), (70, 260, 8, 4, 64, None)])
def test_attention_many_blocks(b, t, h, kv, d, window, dtype):
    """Enough heads that each wave has rows (and keys) of its own; a few of the
    clips are compared, the others against the same clips alone."""
    q, k, v, grad = attention_case(b, t, t, h, kv, d, dtype, 1, packed=True)
    got = attention_run(q, k, v, grad, window)
    pick = [0, b // 2, b - 1]
    part = [x[pick] for x in (q, k, v, grad)]
    check({n: x[pick] for n, x in got.items()}, ref.attention(*part, window, d ** -0.5, None))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,s,window,lengths", [(70, 70, 20, [70, 0, 1, 33, 64]), (70, 70, None, [70, 0, 1, 32, 69]),
                                                (5, 200, None, [200, 195, 196, 198, 0]), (200, 200, 250, [7, 200, 128, 129, 127])])
def test_attention_padding(t, s, window, lengths, dtype):
    """Padding holds NaN and infinities, and none of it is read: outputs and
    gradients of padded positions are zeros."""
    q, k, v, grad = attention_case(len(lengths), t, s, 4, 2, 64, dtype, 2)
    want = ref.attention(q, k, v, grad, window, 0.125, lengths)
    for i, n in enumerate(lengths):
        past = s - t
        for x, junk in ((q, math.nan), (grad, math.inf)):
            x[i, max(0, n - past):] = junk
        k[i, n:], v[i, n:] = math.inf, math.nan
    got = attention_run(q, k, v, grad, window, 0.125, torch.tensor(lengths, dtype=torch.int32, device=DEV))
    check(got, want)
    for i, n in enumerate(lengths):
        assert not got["out"][i, max(0, n - (s - t)):].any() and not got["dq"][i, max(0, n - (s - t)):].any()
        assert not got["dk"][i, n:].any() and not got["dv"][i, n:].any()


def test_attention_lengths_out_of_range_are_clamped():
    q, k, v, grad = attention_case(2, 9, 9, 2, 2, 64, torch.float32, 3)
    got = attention_run(q, k, v, grad, None, None, torch.tensor([-3, 50], dtype=torch.int32, device=DEV))
    check(got, ref.attention(q, k, v, grad, None, 0.125, [0, 9]))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_layouts(dtype):
    """Packed projections, head-major tensors, odd batch strides, expanded
    gradients and unaligned rows give what contiguous copies give."""
    for case in ((2, 50, 50, 4, 2, 64), (1, 50, 50, 4, 4, 32)):
        q, k, v, grad = attention_case(*case, dtype, 4, packed=True)
        want = attention_run(*(x.contiguous() for x in (q, k, v, grad)), 20)
        for name, x in attention_run(q, k, v, grad, 20).items():
            assert torch.equal(x, want[name]), name
        major = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v, grad)]
        for name, x in attention_run(*major, 20).items():
            assert torch.equal(x, want[name]), name
        odd = []
        for x in (q, k, v, grad):
            room = torch.empty(x.numel() + 1, dtype=dtype, device=DEV)[1:].view(x.shape)
            odd.append(room.copy_(x))
        for name, x in attention_run(*odd, 20).items():
            assert torch.equal(x, want[name]), name
        flat = grad[:, :1, :1].expand(grad.shape)
        same = attention_run(q, k, v, flat.contiguous(), 20)
        for name, x in attention_run(q, k, v, flat, 20).items():
            assert torch.equal(x, same[name]), name


def test_attention_scores_far_apart():
    """Scores that differ by hundreds: the running maximum carries them."""
    q, k, v, grad = attention_case(1, 300, 300, 2, 2, 64, torch.float32, 5)
    k = k * torch.linspace(1, 40, 300, device=DEV)[None, :, None, None]
    check(attention_run(q, k, v, grad, None), ref.attention(q, k, v, grad, None, 0.125, None))
    k = k.flip(1)
    check(attention_run(q, k, v, grad, None), ref.attention(q, k, v, grad, None, 0.125, None))


def test_attention_minus_infinity_keys():
    """A key of -inf scores against positive queries takes no probability; rows
    that see nothing else give zeros, as masked ones do."""
    q, k, v, grad = attention_case(1, 40, 40, 1, 1, 64, torch.float32, 6)
    q = q.abs()
    lowest = k.clone()
    lowest[:, :3] = torch.finfo(torch.float32).min / 128
    k[:, :3] = -math.inf
    out, lse = tr.window_attention_forward(q, k, v)
    assert not out[0, :3].any() and (lse[0, :3] == -math.inf).all()
    want, bound = ref.attention(q[:, 3:], k[:, 3:], v[:, 3:], grad[:, 3:], None, 0.125, None)
    ref.assert_within("out", out[:, 3:], want["out"], bound["out"])
    # The type's lowest values are far below every other score and above none.
    out = tr.window_attention_forward(q, lowest, v)[0]
    ref.assert_within("out", out[:, 3:], want["out"], bound["out"])


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_minus_infinity_keys_have_no_gradient(dtype):
    """Probability zero in every row, also beside the rows that fill up a tile."""
    q, k, v, grad = attention_case(1, 40, 40, 2, 1, 64, dtype, 6)
    q = q.abs()
    k[:, :3] = -math.inf
    got = attention_run(q, k, v, grad, None)
    assert not got["dk"][:, :3].any() and not got["dv"][:, :3].any()
    want, bound = ref.attention(q[:, 3:], k[:, 3:], v[:, 3:], grad[:, 3:], None, 0.125, None)
    for n in ("out", "dk", "dv"):
        ref.assert_within(n, got[n][:, 3:], want[n], bound[n])


def test_attention_scores_that_overflow():
    """Scores of -1e42 are minus infinity in FP32: no probability, no gradient, as
    for a key whose score is far below the others but finite."""
    q, k, v, grad = attention_case(1, 80, 80, 2, 2, 64, torch.float32, 10)
    q[..., 0] = 1e21 * (1 + q[..., 0].abs())
    k[..., 0] = 0.0
    low = k.clone()
    k[:, 5, :, 0], low[:, 5, :, 0] = -1e21, -1e-17
    got = attention_run(q, k, v, grad, None)
    assert not got["dk"][:, 5].any() and not got["dv"][:, 5].any()
    check(got, ref.attention(q, low, v, grad, None, 0.125, None))


@pytest.mark.parametrize("b,t,h,kv,pick", [(1, 70, 2, 1, [0]), (40, 160, 8, 8, [0, 39]), (24, 140, 16, 16, [3])])
def test_attention_values_near_the_types_largest(b, t, h, kv, pick):
    """FP32 factors that have no bf16 pieces (2^127 and more) among ordinary ones,
    as a value, a key, a query and a gradient, in blocks of every kind."""
    q, k, v, grad = attention_case(b, t, t, h, kv, 64, torch.float32, 8)
    grad = grad * 1e-3
    for i in pick:
        v[i, 5, 0, 3] = 3.399e38
        v[i, 20, 0, 1] = -2.0 ** 127
    q[pick[0], 9, 0, 2], k[pick[0], :, 0, 2] = 2.0e38, k[pick[0], :, 0, 2] * 1e-38
    got = attention_run(q, k, v, grad, None)
    part = [x[pick] for x in (q, k, v, grad)]
    want, bound = ref.attention(*part, None, 0.125, None)
    most, got = torch.finfo(torch.float32).max, {n: x[pick].double().cpu() for n, x in got.items()}
    for n, x in want.items():
        # dS, near 1e34 through the largest value, times the query 2e38 leaves FP32:
        # what exceeds the type's largest value by more than its bound rounds to infinity.
        over = (x.abs() - ref.SECOND_ORDER * bound[n].expand_as(x) > most) & (n in ("dq", "dk"))
        assert torch.equal(got[n][over], x[over].sign() * math.inf), n
        got[n], want[n] = got[n].masked_fill(over, 0.0), x.masked_fill(over, 0.0)
    check(got, (want, bound))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,t,h,kv,d,window", [(1, 5, 1, 1, 64, 1), (3, 70, 8, 2, 64, 1), (2, 40, 2, 2, 128, 1),
                                               (50, 200, 8, 8, 64, 1), (2, 1, 4, 4, 64, None)])
def test_attention_one_key_has_no_query_gradient(b, t, h, kv, d, window, dtype):
    """One visible key: dP is exactly the row's delta. What is left of dQ is FP32
    rounding: a 16-bit output's own (u |G| |O|) must not reach it, other than times
    the error es of a probability of one."""
    q, k, v, grad = attention_case(b, t, t, h, kv, d, dtype, 12)
    got = attention_run(q, k, v, grad, window)["dq"].double().cpu()
    q, grad = q.double().cpu(), grad.double().cpu()
    k, v = (x.double().cpu().repeat_interleave(h // kv, 2) for x in (k, v))
    size = (grad.abs() * v.abs()).sum(-1, keepdim=True)  # no less than |dP|, |delta|
    es = (d + 8) * ref.H * (q.abs() * k.abs()).sum(-1, keepdim=True) * d ** -0.5
    if dtype == torch.float32:
        ds = 2 * (d + 4) * ref.H * size
    else:  # (1 - p) (dP - delta), and four FP32 roundings of values of that size
        ds = es * 2 * ref.half(dtype) * size + 6 * ref.H * size
    bound = ds * k.abs() * d ** -0.5 * 1.01 + ref.step0(dtype)
    assert (got.abs() <= bound).all(), (got.abs() / bound).max()


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("b,t,h,kv,d,window", [(7, 4, 2, 1, 128, None), (1, 13, 8, 8, 64, None), (16, 2, 4, 4, 64, None),
                                               (3, 30, 4, 2, 32, None), (2, 100, 4, 4, 64, 30)])
def test_attention_gradients_of_few_rows(b, t, h, kv, d, window, dtype):
    """Few keys and few rows: the only 16-bit rounding that counts is the gradients' own."""
    q, k, v, grad = attention_case(b, t, t, h, kv, d, dtype, 13)
    got = attention_run(q, k, v, grad, window)
    del got["out"]
    check(got, ref.attention(q, k, v, grad, window, d ** -0.5, None, pieces=2))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_infinities_reach_what_sees_them(dtype):
    """An infinite key scores minus infinity against positive queries (no
    probability) and an infinite value makes the rows that see it infinite; an
    infinite gradient reaches the keys its row sees. The rows before them, in
    other tiles, are as they were."""
    q, k, v, grad = attention_case(1, 130, 130, 1, 1, 64, dtype, 9)
    q = q.abs()
    clean = attention_run(q, k, v, grad, None)
    v[0, 100, 0, 7] = math.inf
    got = attention_run(q, k, v, grad, None)
    assert torch.equal(got["out"][0, :96], clean["out"][0, :96])
    assert (got["out"][0, 100:, 0, 7] == math.inf).all()
    assert torch.isfinite(got["out"][0, 100:, 0, :7]).all()
    v[0, 100, 0, 7] = 0.0
    grad[0, 3, 0, 2] = math.inf
    got = attention_run(q, k, v, grad, None)
    assert (got["dv"][0, :4, 0, 2] == math.inf).all() and torch.isfinite(got["dv"][0, 64:]).all()


def test_attention_scale_and_window_beyond_the_keys():
    q, k, v, grad = attention_case(1, 60, 60, 2, 2, 64, torch.float32, 7)
    check(attention_run(q, k, v, grad, 10 ** 9, 0.5), ref.attention(q, k, v, grad, None, 0.5, None))


def test_attention_empty():
    for b, t, s in ((0, 5, 5), (2, 0, 5), (2, 0, 0)):
        q, k, v, grad = attention_case(b, t, s, 2, 2, 64, torch.float32)
        got = attention_run(q, k, v, grad, None)
        assert got["out"].shape == q.shape and not got["dk"].any() and not got["dv"].any()


def test_attention_far_rows():
    """A cache whose rows lie more than 2^31 elements from its base."""
    s, pitch = 600, 4_000_000
    base = torch.empty(s * pitch, dtype=torch.float16, device=DEV)
    q, k, v, grad = attention_case(1, 300, s, 2, 1, 64, torch.float16, 8)
    far = []
    for i, x in enumerate((k, v)):
        view = base.as_strided((1, s, 1, 64), (0, pitch, 64, 1), 64 * i)
        far.append(view.copy_(x))
    want = attention_run(q, k, v, grad, 400)
    for name, x in attention_run(q, *far, grad, 400).items():
        assert torch.equal(x, want[name]), name


def test_attention_repeats_bit_for_bit():
    q, k, v, grad = attention_case(2, 333, 333, 8, 2, 64, torch.bfloat16, 9)
    first = attention_run(q, k, v, grad, 100)
    for _ in range(3):
        for name, x in attention_run(q, k, v, grad, 100).items():
            assert torch.equal(x, first[name]), name


# ------------------------------------------------------- codebook embedding
def embedding_case(b, books, frames, entries, dim, dtype, seed=0, skew=False):
    g = gen(seed)
    codes = torch.randint(-1, entries, (b, books, frames), generator=g)
    if skew:
        codes = torch.where(torch.rand(codes.shape, generator=g) < 0.6, min(3, entries - 1), codes)
    table = torch.randn(books, entries, dim, generator=g).to(dtype)
    return codes.to(DEV), table.to(DEV), torch.randn(b, frames, dim, generator=g).to(dtype).to(DEV)


def embedding_run(codes, table, grad, scale):
    return {"out": tr.code_embedding_forward(codes, table, scale),
            "dtable": tr.code_embedding_backward(grad, codes, table, scale)}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,books,frames,entries,dim", [(1, 1, 1, 1, 8), (1, 8, 13, 2048, 256), (3, 4, 40, 16, 64), (2, 9, 77, 300, 200),
                                                        (1, 2, 700, 2049, 24), (2, 3, 50, 9000, 17), (1, 1, 3000, 5, 1024)])
@pytest.mark.parametrize("skew", [False, True])
def test_embedding(b, books, frames, entries, dim, skew, dtype):
    codes, table, grad = embedding_case(b, books, frames, entries, dim, dtype, 0, skew)
    check(embedding_run(codes, table, grad, 1.7), ref.embedding(codes, table, grad, 1.7))


def test_embedding_one_code_owns_everything():
    codes, table, grad = embedding_case(2, 2, 5000, 64, 128, torch.float32, 1)
    codes[:, 0] = 63
    codes[:, 1] = 0
    check(embedding_run(codes, table, grad, -0.5), ref.embedding(codes, table, grad, -0.5))


def test_embedding_all_absent():
    codes, table, grad = embedding_case(2, 2, 50, 64, 128, torch.float32, 2)
    codes[:] = -1
    got = embedding_run(codes, table, grad, 2.0)
    assert not got["out"].any() and not got["dtable"].any()


def test_embedding_bad_codes_are_nan_and_take_no_gradient():
    codes, table, grad = embedding_case(2, 3, 20, 50, 64, torch.float32, 3)
    want = ref.embedding(codes.masked_fill(torch.eye(20, device=DEV).bool()[None, [2, 5, 7]], -1), table, grad, 1.0)
    for j, (t, bad) in enumerate(((2, 50), (5, -2), (7, 1 << 40))):
        codes[:, j, t] = bad
    got = embedding_run(codes, table, grad, 1.0)
    assert got["out"][:, [2, 5, 7]].isnan().all()
    rest = [t for t in range(20) if t not in (2, 5, 7)]
    assert torch.isfinite(got["out"][:, rest]).all()
    ref.assert_within("dtable", got["dtable"], want[0]["dtable"], want[1]["dtable"])


def test_embedding_views():
    """Codebook slices (the split quantizer's two sums), a strided frame axis,
    a gradient slice."""
    codes, table, grad = embedding_case(3, 8, 30, 64, 128, torch.float32, 4)
    wide = torch.randn(3, 30, 300, generator=gen(5)).to(DEV)
    for c, t, g in ((codes[:, 1:], table[1:], wide[..., 4:132]), (codes[:, :1], table[:1], wide[..., 3:131]),
                    (codes.transpose(1, 2).contiguous().transpose(1, 2), table, grad.transpose(0, 1).contiguous().transpose(0, 1))):
        check(embedding_run(c, t, g, 1.0), ref.embedding(c, t, g, 1.0))


def test_embedding_matches_the_decoders_sum():
    """One codebook set at scale 1 is the decoder's own gather-sum, bit for bit."""
    from fast_mimi_amd import ops

    codes, table, _ = embedding_case(2, 8, 33, 2048, 256, torch.float32, 6)
    codes = codes.clamp(min=0)
    out = torch.empty(2 * 33, 512, device=DEV)
    ops.call("fm_rvq_decode", codes, 2, 8, 33, 1, table, 2048, 256, out)
    out = out.view(2, 33, 512)
    assert torch.equal(tr.code_embedding_forward(codes[:, :1], table[:1]), out[..., :256])
    assert torch.equal(tr.code_embedding_forward(codes[:, 1:], table[1:]), out[..., 256:])


def test_embedding_table_may_change_before_the_backward_pass():
    codes, table, grad = embedding_case(2, 3, 40, 32, 64, torch.float32, 8)
    table.requires_grad_()
    out = tr.code_embedding(codes, table)
    with torch.no_grad():
        table.mul_(2.0)
    out.backward(grad)
    assert torch.equal(table.grad, tr.code_embedding_backward(grad, codes, table))


def test_embedding_far_entries():
    """Codebooks of more than 2^31 elements."""
    books, entries, dim = 5, 32768, 13200
    table = torch.zeros(books, entries, dim, dtype=torch.float16, device=DEV)
    assert table.numel() > 1 << 31
    table[4, -1] = torch.arange(dim, device=DEV) % 100
    codes = torch.full((1, books, 3), entries - 1, device=DEV)
    assert torch.equal(tr.code_embedding_forward(codes, table)[0, 1], table[4, -1])
    grad = (torch.arange(3, device=DEV)[None, :, None] + 1).expand(1, 3, dim).half()
    dtable = tr.code_embedding_backward(grad, codes, table)
    assert (dtable[:, -1] == 6).all() and not dtable[:, :64].any() and not dtable[4, -64:-1].any()


def test_embedding_repeats_bit_for_bit():
    codes, table, grad = embedding_case(4, 4, 3000, 100, 256, torch.float32, 7, True)
    first = tr.code_embedding_backward(grad, codes, table)
    for _ in range(3):
        assert torch.equal(tr.code_embedding_backward(grad, codes, table), first)


# ------------------------------------------------ autograd, together, captured
def model(codes, table, w, b, proj, window, lengths, f):
    """Codes through one attention layer to a loss: the operators as a
    transformer over the codes uses them, with ``f`` theirs or the definition's."""
    x = f.code_embedding(codes, table, 0.5)
    y = f.layer_norm(x, w, b)
    n, t, c = y.shape
    qkv = (y @ proj).view(n, t, 3 * c)
    heads = c // 64
    q, k, v = (qkv[..., i * c:(i + 1) * c].reshape(n, t, heads, 64) for i in range(3))
    z = f.window_attention(q, k, v, window, None, lengths).reshape(n, t, c)
    z = f.layer_norm(x + z, w, b)
    return (z * z.tanh()).sum()


class Definition:
    """The same operators as torch formulas, differentiated by autograd."""

    @staticmethod
    def code_embedding(codes, table, scale):
        at = codes.clamp(min=0)
        picked = torch.stack([table[j][at[:, j]] for j in range(table.shape[0])], 1)
        return scale * (picked * (codes >= 0)[..., None]).sum(1)

    @staticmethod
    def layer_norm(x, w, b):
        return torch.nn.functional.layer_norm(x, x.shape[-1:], w, b, 1e-5)

    @staticmethod
    def window_attention(q, k, v, window, scale, lengths):
        n, t, h, d = q.shape
        see = torch.stack([ref.visible(t, t, window, t if lengths is None else int(lengths[i])) for i in range(n)])[:, None]
        s = (q.transpose(1, 2) @ k.transpose(1, 2).transpose(2, 3)) * d ** -0.5
        live = see.any(-1, keepdim=True)
        p = torch.softmax(s.masked_fill(~see, -math.inf).masked_fill(~live, 0.0), -1) * live
        return (p @ v.transpose(1, 2)).transpose(1, 2)


def model_case(dtype=torch.float32, seed=0):
    g = gen(seed)
    codes = torch.randint(-1, 64, (3, 4, 40), generator=g)
    table = torch.randn(4, 64, 128, generator=g)
    w, b = 1 + 0.1 * torch.randn(128, generator=g), 0.1 * torch.randn(128, generator=g)
    proj = torch.randn(128, 384, generator=g) / 8
    return codes, [t.to(dtype) for t in (table, w, b, proj)], torch.tensor([40, 17, 3], dtype=torch.int32)


def test_operators_together_against_the_definition():
    """Codes -> embedding -> LayerNorm -> attention -> LayerNorm, differentiated
    through autograd, against the same in 64 bits.  Each of the eight steps adds
    errors of FP32 sums of at most 384 terms (random signs: about 20 H each) and
    passes on those before, amplified by at most a few: 1e-5 of a gradient's norm."""
    codes, params, lengths = model_case()
    leaves = [p.to(DEV).requires_grad_() for p in params]
    loss = model(codes.to(DEV), *leaves, 16, lengths.to(DEV), tr)
    got = torch.autograd.grad(loss, leaves)
    wide = [p.double().requires_grad_() for p in params]
    want_loss = model(codes, *wide, 16, lengths, Definition)
    want = torch.autograd.grad(want_loss, wide)
    assert abs(loss.item() - want_loss.item()) <= 1e-5 * abs(want_loss.item())
    for a, e in zip(got, want):
        assert (a.double().cpu() - e).norm() <= 1e-5 * e.norm()


def test_gradients_against_differences():
    """Directional derivatives of the 64-bit definition by central differences
    (step 1e-5: an error of 1e-10 of the third derivative and 1e-11 of the
    value) equal the operators' gradients in that direction, to their FP32 error."""
    codes, params, lengths = model_case(seed=1)
    leaves = [p.to(DEV).requires_grad_() for p in params]
    got = torch.autograd.grad(model(codes.to(DEV), *leaves, 16, lengths.to(DEV), tr), leaves)
    g = gen(2)
    for i, p in enumerate(params):
        direction = torch.randn(p.shape, generator=g, dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            moved = [x.double() for x in params]
            moved[i] = moved[i] + sign * 1e-5 * direction
            ends.append(model(codes, *moved, 16, lengths, Definition).item())
        slope = (ends[0] - ends[1]) / 2e-5
        along = (got[i].double().cpu() * direction).sum().item()
        assert abs(along - slope) <= 1e-5 * got[i].double().norm().item() * direction.norm().item()


def test_needs_of_each_input():
    """Only asked-for gradients come back; inputs without any give no graph."""
    q, k, v, grad = attention_case(1, 10, 10, 2, 2, 64, torch.float32)
    full = attention_run(q, k, v, grad, None)
    k.requires_grad_()
    (dk,) = torch.autograd.grad(tr.window_attention(q, k, v), (k,), grad)
    assert torch.equal(dk, full["dk"])
    assert not tr.window_attention(q, k.detach(), v).requires_grad
    with torch.no_grad():
        assert not tr.window_attention(q, k, v).requires_grad


def test_second_derivatives_are_refused():
    x = torch.randn(4, 64, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(tr.layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_inputs_changed_before_backward_are_refused():
    q, k, v, grad = attention_case(1, 10, 10, 2, 2, 64, torch.float32)
    a = q.clone().requires_grad_()
    out = tr.window_attention(a, k, v)
    k.mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        out.backward(grad)


def test_negated_views():
    """Lazily negated inputs are what they stand for."""
    x, grad, w, b = norm_case(6, 64, torch.float32, torch.float32, 7)
    neg = torch._neg_view(x)
    assert neg.is_neg()
    assert torch.equal(tr.layer_norm_forward(neg, w, b)[0], tr.layer_norm_forward(-x, w, b)[0])


def step(state):
    """One training step without autograd, everything it computes."""
    codes, table, w, b, q, k, v, grad, lengths = state
    x = tr.code_embedding_forward(codes, table, 0.5)
    y, mean, rstd = tr.layer_norm_forward(x, w, b)
    dx, dw, db = tr.layer_norm_backward(x, x, mean, rstd, w, b)
    dtable = tr.code_embedding_backward(dx, codes, table, 0.5)
    out, lse = tr.window_attention_forward(q, k, v, 50, None, lengths)
    return [x, y, dx, dw, db, dtable, out, *tr.window_attention_backward(grad, q, k, v, out, lse, 50, None, lengths)]


def step_state(seed, dtype=torch.bfloat16):
    codes, table, _ = embedding_case(2, 4, 300, 64, 128, dtype, seed, True)
    _, _, w, b = norm_case(1, 128, dtype, dtype, seed)
    q, k, v, grad = attention_case(2, 2, 900, 4, 2, 64, dtype, seed)
    return [codes, table, w, b, q, k, v, grad, torch.tensor([900, 899], dtype=torch.int32, device=DEV)]


def test_captured_steps_share_nothing():
    """Two graphs of the same step on inputs of their own, replayed in turn with
    eager work between, new inputs copied in: each replay equals the eager call."""
    static = [step_state(1), step_state(2)]
    for s in static:
        step(s)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(s))
        graphs.append(g)
    for turn in range(4):
        for i in (0, 1):
            for to, fresh in zip(static[i], step_state(10 + 2 * turn + i)):
                to.copy_(fresh)
        graphs[0].replay()
        graphs[1].replay()
        want = [step(s) for s in static]
        torch.cuda.synchronize()
        for got, expected in zip(outs, want):
            for x, y in zip(got, expected):
                assert torch.equal(x, y)


def test_on_another_stream():
    """Calls run on the current stream, whichever that is."""
    state = step_state(3)
    want = step(state)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(10_000_000)
        fresh = [x.clone() for x in state]
        got = step(fresh)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_captured_backward_of_a_leaf_in_an_eager_graph_is_refused():
    x = torch.randn(8, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    y = tr.layer_norm(x, w)  # its graph stays alive
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        with torch.cuda.graph(g):
            tr.layer_norm(x, w)
    # Without it the same step is captured and replays.
    del y
    ones = torch.ones(8, 64, device=DEV)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = tr.layer_norm(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), ones)
    with torch.no_grad():
        x.copy_(torch.randn(8, 64, device=DEV))
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, tr.layer_norm_forward(x.detach(), w.detach())[0])


def test_operators_are_traced_as_mutating_calls():
    """``torch.ops.fast_mimi_amd`` has the same entry points."""
    x, grad, w, b = norm_case(6, 64, torch.float32, torch.float32, 8)
    y, mean, rstd = torch.empty_like(x), torch.empty(6, device=DEV), torch.empty(6, device=DEV)
    torch.ops.fast_mimi_amd.layer_norm_forward(x, 64, w, b, 6, 64, 1e-5, 0, 0, y, mean, rstd)
    assert torch.equal(y, tr.layer_norm_forward(x, w, b)[0])
