"""The operators of quantised and differential transformers on the GPU, against their definitions in float64.

Tolerances count roundings. U = 2^-24 is half a step of float32, HALF[T] half a step of the arrays' type; results of float16 below its normal range are
off by up to 2^-25 on top."""
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

import dace_onnx_amd.onnx as donnx
from dace_onnx_amd import _lib
from dace_onnx_amd.onnx.proto import helper, numpy_helper
import llm_operators as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, F16, BF = R.TYPES
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF: 2.0 ** -134}


def normal(seed, *shape, scale=1.0, dtype=F32):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def within(got, expected, bound):
    """|got - expected| <= bound, element by element; nothing else is finite."""
    assert got.shape == expected.shape
    error = (got.double() - expected).abs()
    worst = (error / bound).max().item() if got.numel() else 0.0
    assert worst <= 1, f"{worst:.3g} of the bound; largest error {error.max().item():.3g}"


# ---------------------------------------------------------------------------------------------- SkipRMSNormalization
# The sum of squares is a chain of at most 64 fused multiply-adds in a thread (of a long row: cols / 1024) and 16 additions across threads, all of
# positive numbers; its relative error halves under the square root. The sum with the residual, the division by the number of columns, the root, the
# reciprocal and two products are a rounding each, 2^-23 for the root and the reciprocal.


def norm_bound(columns):
    return (max(64, columns / 1024) + 16) / 2 * U + 10 * U


def check_norm(x, gain, skip, y, total, q, scale, epsilon=1e-5):
    dtype, b = x.dtype, norm_bound(x.shape[-1])
    ey, es, _, escale = R.rms_norm(x, gain, skip, epsilon)
    if y is not None:
        assert y.dtype == dtype
        within(y, ey, (R.HALF[dtype] + b * (1 + R.HALF[dtype])) * ey.abs() + TINY[dtype])
    if total is not None:
        within(total, es, (R.HALF[dtype] + U) * es.abs() + TINY[dtype])
    if q is not None:
        assert q.dtype == torch.int8 and scale.dtype == F32
        within(scale, escale, (b + U) * escale + 2.0 ** -149)
        ratio = ey / torch.where(escale > 0, escale, 1.0)[..., None]
        within(q, ratio, 0.5 + 2 * 127 * (b + 2 * U) + 0 * ratio)   # half a step, and what y and the scale are off by
        assert torch.equal(q.abs().amax(-1).to(torch.int32), torch.where(escale > 0, 127, 0).to(torch.int32))


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("rows, columns", [(1, 1), (1, 64), (3, 7), (5, 255), (2, 256), (4, 257), (9, 512), (3, 1001), (2, 2048), (7, 2049), (3, 4097), (2, 8192),
                                           (2, 10007), (1, 16384), (2, 16385), (1, 32768), (3, 32769), (1, 70001), (1030, 96)])
def test_norm(dtype, rows, columns):
    x, skip, gain = normal(1, rows, columns, scale=3, dtype=dtype), normal(2, rows, columns, dtype=dtype), normal(3, columns, scale=0.5, dtype=dtype) + 1
    shape = (rows, columns)
    outs = [("y", dtype, shape), ("s", dtype, shape), ("q", torch.int8, shape), ("qs", F32, (rows,))]
    check_norm(x, gain, skip, *R.call("SkipRMSNormalization", [("x", x), ("g", gain), ("skip", skip)], outs))
    q, scale = R.call("SkipRMSNormalization", [("x", x), ("g", gain), ("skip", None)], [None, None, *outs[2:]], epsilon=0.5)
    check_norm(x, gain, None, None, None, q, scale, 0.5)


def test_norm_over_several_dimensions():
    x, gain = normal(4, 2, 3, 5, 8), normal(5, 5, 8)
    y, q, scale = R.call("SkipRMSNormalization", [("x", x), ("g", gain), ("skip", None)],
                         [("y", F32, x.shape), None, ("q", torch.int8, x.shape), ("qs", F32, (2, 3))], axis=2)
    check_norm(x.reshape(6, 40), gain.reshape(40), None, y.reshape(6, 40), None, q.reshape(6, 40), scale.reshape(6))


def test_norm_of_many_rows():
    """2^22 rows and more, as the heads of long prompts are."""
    rows, columns = (1 << 22) + 5, 8
    x, gain = normal(1, rows, columns, dtype=BF), normal(2, columns, dtype=BF)
    check_norm(x, gain, None, *R.call("SkipRMSNormalization", [("x", x), ("g", gain), ("skip", None)], [("y", BF, x.shape), None, ("q", torch.int8, x.shape), ("qs", F32, (rows,))])[:1],
               None, None, None)


@pytest.mark.parametrize("columns", [40, 300, 40000])
def test_norm_of_extreme_rows(columns):
    """Squares beyond float32, squares that vanish in it, rows of zeros, rows with an infinity or a NaN."""
    x = normal(6, 7, columns)
    for row, factor in enumerate((1e30, 2.0 ** 100, 1e-30, 1e-38, 0.0)):
        x[row] *= factor
    x[5, 3], x[6, columns - 1] = torch.inf, torch.nan
    gain = normal(7, columns)
    outs = [("y", F32, x.shape), None, ("q", torch.int8, x.shape), ("qs", F32, (7,))]
    for epsilon in (1e-6, 0.0):
        y, q, scale = R.call("SkipRMSNormalization", [("x", x), ("g", gain), ("skip", None)], outs, epsilon=epsilon)
        finite = slice(0, 5) if epsilon else slice(0, 4)   # zeros without epsilon are 0 / 0
        check_norm(x[finite], gain, None, y[finite], None, q[finite], scale[finite], epsilon)
        assert scale[finite.stop:].isnan().all() and (q[finite.stop:] == 0).all()
        assert y[5, 3].isnan() and y[6].isnan().all()
        if epsilon:
            assert scale[4] == 0 and (y[4] == 0).all()
        else:
            assert y[4].isnan().all()


@pytest.mark.parametrize("columns", [40, 300, 16000, 40000])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_norm_of_rows_at_the_ends_of_the_exponents(columns, dtype):
    """Rows whose values are the largest that there are, one such value among ones, and the smallest."""
    x = normal(6, 4, columns).clamp(-3.9, 3.9)
    x = torch.stack([x[0].sign() * torch.finfo(dtype).max, x[1] * 2.0 ** 126, x[2], x[3] * 2.0 ** -130]).to(dtype)
    x[2, 7] = -torch.finfo(dtype).max
    gain = normal(7, columns, dtype=dtype)
    y, q, scale = R.call("SkipRMSNormalization", [("x", x), ("g", gain), ("skip", None)], [("y", dtype, x.shape), None, ("q", torch.int8, x.shape), ("qs", F32, (4,))], epsilon=0.0)
    check_norm(x, gain, None, y, None, q, scale, 0.0)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("columns", [5, 24, 777, 9000])
def test_norm_at_any_address_and_over_its_input(dtype, columns):
    lib, rows = _lib.library(), 6
    buffers = [torch.zeros(rows * columns + 9, dtype=dtype, device="cuda") for _ in range(5)]
    x, skip, gain, y, total = (b[i + 1:i + 1 + rows * columns].view(rows, columns) for i, b in enumerate(buffers))   # odd addresses, each another
    gain = gain.reshape(-1)[:columns]
    x.copy_(normal(8, rows, columns, dtype=dtype)), skip.copy_(normal(9, rows, columns, dtype=dtype)), gain.copy_(normal(10, columns, dtype=dtype))
    q, scale = torch.zeros(rows * columns + 9, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
    q8 = q[3:3 + rows * columns].view(rows, columns)
    run = lambda y, s: _lib.check(lib.mi355x_skip_rms_norm(x.data_ptr(), skip.data_ptr(), gain.data_ptr(), y.data_ptr(), s.data_ptr(), q8.data_ptr(),  # noqa: E731
                                                          scale.data_ptr(), rows, columns, R.ELEMENT[dtype], 1e-5, _lib.current_stream()), "norm")
    run(y, total)
    check_norm(x, gain, skip, y, total, q8, scale)
    assert all(b[:i + 1].abs().max() == 0 and b[i + 1 + rows * columns:].abs().max() == 0 for i, b in enumerate(buffers) if i != 2)
    assert q[:3].abs().max() == 0 and q[3 + rows * columns:].abs().max() == 0
    first = x.clone(), y.clone(), total.clone(), q8.clone()
    run(skip, x)   # the sum over x, the norm over the residual
    assert torch.equal(x, first[2]) and torch.equal(skip, first[1]) and torch.equal(q8, first[3])


# ---------------------------------------------------------------------------------------------- QuantizedLinear
# The sum is exact. Its conversion, two scales, the bias and the residual are a rounding each, at most U of the magnitudes that are added; erf and exp
# are off by up to 2 U absolutely, times at most the value, the exponent's rounding moves silu by at most v^2 e^v / (1 + e^v)^2 U < U, Gelu's and Silu's slopes
# stay below 1.13, the division and products around them add 4 U.


def linear_bound(size, expected, dtype):
    return 16 * U * (size + 1) + R.HALF[dtype] * expected.abs() + TINY[dtype]


def eight(seed, *shape):
    return torch.randint(-128, 128, shape, generator=torch.Generator().manual_seed(seed), dtype=torch.int32).to(torch.int8).cuda()


@pytest.mark.parametrize("m, n, k", [(1, 1, 1), (1, 16, 64), (2, 17, 15), (3, 40, 16), (16, 33, 130), (17, 64, 128), (31, 65, 1000), (33, 129, 1025), (64, 256, 512), (65, 48, 2048),
                                     (130, 260, 96), (197, 201, 333), (256, 256, 256), (300, 515, 384), (513, 300, 640), (5, 1000, 4096), (260, 1030, 1024), (1100, 530, 64),
                                     (40, 24, 0), (128, 128, 131071)])
@pytest.mark.parametrize("dtype", R.TYPES)
def test_linear(m, n, k, dtype):
    x, w = eight(1, m, k), eight(2, n, k)
    xs, ws = normal(3, m).abs() / 74 + 1e-3, normal(4, n).abs() / 74 / max(k, 1) ** 0.5
    bias, residual = normal(5, n, dtype=dtype), normal(6, m, n, dtype=dtype)
    for i, activation in enumerate(_lib.ACTIVATIONS):
        b, r = bias if i & 1 else None, residual if i & 2 else None
        y, = R.call("QuantizedLinear", [("x", x), ("w", w), ("xs", xs), ("ws", ws), ("b", b), ("r", r)], [("y", dtype, (m, n))], activation=activation, to=R.ELEMENT[dtype])
        expected, size = R.quantized_linear(x, w, xs, ws, b, r, activation)
        assert y.dtype == dtype
        within(y, expected, linear_bound(size, expected, dtype))


@pytest.mark.parametrize("form", range(5))
@pytest.mark.parametrize("m, n, k", [(1, 1, 1), (63, 65, 16), (65, 63, 127), (129, 140, 128), (300, 270, 144), (257, 129, 272), (64, 513, 1009), (515, 40, 640), (7, 9, 0)])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_linear_by_every_kernel(form, m, n, k, dtype, tuning):
    x, w, xs, ws = eight(1, m, k), eight(2, n, k), normal(3, m).abs() / 74 + 1e-3, normal(4, n).abs() / 74 / max(k, 1) ** 0.5
    bias, residual = normal(5, n, dtype=dtype), normal(6, m, n, dtype=dtype)
    tuning(MI355X_QLIN_FORM=form)
    y, = R.call("QuantizedLinear", [("x", x), ("w", w), ("xs", xs), ("ws", ws), ("b", bias), ("r", residual)], [("y", dtype, (m, n))], activation="gelu", to=R.ELEMENT[dtype])
    expected, size = R.quantized_linear(x, w, xs, ws, bias, residual, "gelu")
    within(y, expected, linear_bound(size, expected, dtype))


def test_linear_with_one_scale_and_more_dimensions():
    x, w = eight(1, 2, 3, 70), eight(2, 50, 70)
    y, = R.call("QuantizedLinear", [("x", x), ("w", w), ("xs", normal(3, 1).abs()), ("ws", normal(4, 1).abs())], [("y", F32, (2, 3, 50))])
    expected, size = R.quantized_linear(x.reshape(6, 70), w, normal(3, 1).abs().expand(6), normal(4, 1).abs().expand(50))
    within(y.reshape(6, 50), expected, linear_bound(size, expected, F32))


@pytest.mark.parametrize("k", [17, 18, 19, 127, 129, 130, 131, 133, 1155, 2049, 4091, 4094, 4095])
@pytest.mark.parametrize("m, n", [(1, 1), (5, 33), (70, 40)])
def test_linear_straight_from_memory_of_odd_rows(m, n, k, tuning):
    """Arrays that begin at words and rows that do not, arrays that do not; what lies before and behind them would change the sums."""
    tuning(MI355X_QLIN_FORM=0)
    lib = _lib.library()
    for front in (4, 3):
        x, w = (torch.cat([t.new_full((front,), 127), t.reshape(-1), t.new_full((32,), 127)]) for t in (eight(1, m, k), eight(2, n, k)))
        y, one = torch.zeros(m, n, device="cuda"), torch.ones(1, device="cuda")
        _lib.check(lib.mi355x_quantized_linear(x[front:].data_ptr(), w[front:].data_ptr(), one.data_ptr(), one.data_ptr(), None, None, y.data_ptr(), m, n, k, 1, 1, 0, 1, _lib.current_stream()),
                   "linear")
        expected = x[front:front + m * k].view(m, k).double() @ w[front:front + n * k].view(n, k).double().t()
        within(y, expected, U * expected.abs() + TINY[F32])


@pytest.mark.parametrize("k", [16, 17])
def test_linear_of_more_than_32_bits_of_results(k):
    m, n = (1 << 17) + 3, (1 << 14) + 24
    x, w, xs, ws = eight(1, m, k), eight(2, n, k), normal(3, m).abs() / 74 + 1e-3, normal(4, n).abs() / 74
    y, = R.call("QuantizedLinear", [("x", x), ("w", w), ("xs", xs), ("ws", ws)], [("y", F16, (m, n))], to=R.ELEMENT[F16])
    for rows in (slice(0, 300), slice(m // 2, m // 2 + 300), slice(m - 300, m)):
        expected, size = R.quantized_linear(x[rows], w, xs[rows], ws)
        within(y[rows], expected, linear_bound(size, expected, F16))


@pytest.mark.parametrize("m", [2, 300])
@pytest.mark.parametrize("dtype", R.TYPES)
def test_linear_small_results_of_silu(m, dtype):
    """Silu of -1 to -87, exact before it, with errors relative to the results: in float32 of the exponential, the sum and the division 2 U each, in 16 bits |v| U more."""
    n, k = 88, 32
    x, w = torch.full((m, k), -1, dtype=torch.int8, device="cuda"), torch.zeros(n, k, dtype=torch.int8, device="cuda")
    w[:, 0] = torch.arange(n)
    one = torch.ones(1, device="cuda")
    y, = R.call("QuantizedLinear", [("x", x), ("w", w), ("xs", one), ("ws", one)], [("y", dtype, (m, n))], activation="silu", to=R.ELEMENT[dtype])
    v = -torch.arange(n).cuda().double().expand(m, n)
    expected = v / (1 + torch.exp(-v))
    within(y, expected, ((8 + (0 if dtype == F32 else 2) * v.abs()) * U + R.HALF[dtype]) * expected.abs() + TINY[dtype])


@pytest.mark.parametrize("m", [2, 40, 300])
def test_linear_largest_sums_and_scales_that_are_not_numbers(m):
    k = (1 << 17) - 1
    x, w = torch.full((m, k), -128, dtype=torch.int8, device="cuda"), torch.full((20, k), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    xs, ws = torch.ones(m, device="cuda"), torch.ones(20, device="cuda")
    xs[1], ws[3] = torch.nan, torch.inf
    for activation in _lib.ACTIVATIONS:
        y, = R.call("QuantizedLinear", [("x", x), ("w", w), ("xs", xs), ("ws", ws)], [("y", F32, (m, 20))], activation=activation)
        assert y[1].isnan().all() and y[0, 3] == torch.inf
        assert y[0, 0] == 16384 * k   # (of 31 bits, the last 14 zero: a float32)
        if activation == "none":
            assert y[0, 1] == np.float32(-16256 * k)


@pytest.mark.parametrize("m, n, k", [(3, 50, 129), (100, 70, 256), (300, 300, 128)])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_linear_at_any_address_and_into_its_residual(m, n, k, dtype):
    lib = _lib.library()
    x, w = (torch.cat([t.new_zeros(o), t.reshape(-1), t.new_zeros(9)]) for t, o in ((eight(1, m, k), 3), (eight(2, n, k), 5)))
    y, bias = torch.zeros(m * n + 9, dtype=dtype, device="cuda"), torch.cat([torch.zeros(1, dtype=dtype, device="cuda"), normal(5, n, dtype=dtype)])[1:]
    out = y[1:1 + m * n].view(m, n)
    out.copy_(normal(6, m, n, dtype=dtype))
    residual, xs, ws = out.clone(), normal(3, m).abs(), normal(4, n).abs() / k
    _lib.check(lib.mi355x_quantized_linear(x[3:].data_ptr(), w[5:].data_ptr(), xs.data_ptr(), ws.data_ptr(), bias.data_ptr(), out.data_ptr(), out.data_ptr(), m, n, k, m, n, 3,
                                           R.ELEMENT[dtype], _lib.current_stream()), "linear")
    expected, size = R.quantized_linear(x[3:3 + m * k].view(m, k), w[5:5 + n * k].view(n, k), xs, ws, bias, residual, "silu")
    within(out, expected, linear_bound(size, expected, dtype))
    assert y[0] == 0 and y[1 + m * n:].abs().max() == 0


# ---------------------------------------------------------------------------------------------- RotaryPositions
# The angle is right to float64 until it lies within half a turn, as t = 2 / turn in float32: off by U, pi U as an angle; sine and cosine are off by up
# to 2 U more. Two products and their sum are a rounding each, all relative to |a| + |b|.


def rotary_bound(x, expected, dtype):
    return (math.pi + 2 + 2) * U * 2 * x.double().abs().amax(-1, keepdim=True) + R.HALF[dtype] * expected.abs() + TINY[dtype]


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("b, s, h, kv, d, sections", [(1, 1, 1, 0, 2, [1]), (2, 3, 4, 2, 64, [32]), (2, 5, 3, 1, 64, [8, 12, 12]), (1, 37, 2, 2, 80, [5, 7, 9]), (3, 9, 5, 1, 128, [16, 24, 24]),
                                                      (1, 130, 1, 1, 96, [20, 0, 18]), (2, 7, 3, 0, 33, [7, 3]), (1, 3, 2, 1, 256, [128]), (1, 4, 40, 8, 32, [2] * 8), (2, 3, 2, 1, 8, [0])])
def test_rotary(dtype, interleaved, b, s, h, kv, d, sections):
    q, k = normal(1, b, s, h, d, dtype=dtype), normal(2, b, s, kv, d, dtype=dtype) if kv else None
    positions = torch.randint(-70000, 1 << 20, (len(sections), b, s), generator=torch.Generator().manual_seed(3)).cuda()
    frequencies = (10000.0 ** (-torch.arange(sum(sections)) / max(sum(sections), 1))).cuda()
    for p in (positions, positions.to(torch.int32)):
        outs = R.call("RotaryPositions", [("q", q), ("p", p), ("f", frequencies), ("k", k)],
                      [("qo", dtype, q.shape), ("ko", dtype, k.shape) if kv else None], sections=sections, interleaved=interleaved)
        for x, y in zip((q, k), outs):
            expected = R.rotary(x, positions, frequencies, sections, interleaved)
            within(y, expected, rotary_bound(x, expected, dtype))
            assert torch.equal(y[..., 2 * sum(sections):], x[..., 2 * sum(sections):])


def test_rotary_far_positions_and_copied_bits():
    """Positions of 2^40, where float32 would know nothing of the angle; NaN among the values that are not turned."""
    q = normal(1, 1, 2, 2, 24)
    q[..., 16:] = torch.nan
    positions, frequencies = torch.tensor([[[(1 << 40) + 1, -(1 << 40)]]]).cuda(), torch.full((8,), 0.73).cuda()
    y, = R.call("RotaryPositions", [("q", q), ("p", positions), ("f", frequencies), ("k", None)], [("qo", F32, q.shape), None])
    # the angle in fractions: 2^37 turns are off by 2^-16 in float64 and by 2^-16 through 1 / pi, together 2e-4 as an angle
    f = np.float32(0.73)
    for i, p in enumerate(((1 << 40) + 1, -(1 << 40))):
        turns = Fraction(p) * Fraction(float(f)) / (2 * Fraction(math.pi))
        angle = float((turns - round(turns)) * 2) * math.pi
        a, b = q[0, i, 0, 0].item(), q[0, i, 0, 8].item()
        assert abs(y[0, i, 0, 0].item() - (a * math.cos(angle) - b * math.sin(angle))) < 2e-3 * (abs(a) + abs(b))
    assert y[..., 16:].isnan().all()


@pytest.mark.parametrize("dtype", [F32, F16])
def test_rotary_at_any_address_and_over_its_input(dtype):
    lib, (s, h, d) = _lib.library(), (11, 3, 48)
    buffer = torch.zeros(s * h * d + 9, dtype=dtype, device="cuda")
    x = buffer[1:1 + s * h * d].view(1, s, h, d)
    x.copy_(normal(1, 1, s, h, d, dtype=dtype))
    positions, frequencies = torch.arange(s).reshape(1, 1, s).cuda(), normal(2, 16).abs()
    expected, before = R.rotary(x, positions, frequencies, [16], False), x.clone()
    _lib.check(lib.mi355x_rotary_positions(x.data_ptr(), None, positions.data_ptr(), frequencies.data_ptr(), x.data_ptr(), None, s, h, 0, d, 32, 1, _lib.i64_array([16]), 0, 8,
                                           R.ELEMENT[dtype], _lib.current_stream()), "rotary")
    within(x, expected, rotary_bound(before, expected, dtype))
    assert buffer[0] == 0 and buffer[1 + s * h * d:].abs().max() == 0


# ---------------------------------------------------------------------------------------------- DifferentialAttention
# size = sum_j (P1 + |l| P2) |V|. A score is a sum of d products in float32: off by (d + 2) U sum |q k| scale, and by 3 U of its largest magnitude in the base of
# two; P is off by twice that relatively (numerator and sum). The sums over the keys are off by up to Sk U each and by as much again where splits are joined,
# P is rounded to 16 bits where the arrays have them. l is a sum of a few exponentials of short dot products: 8 (vector + 8) U of it.


def attention_bound(q, k, size, expected, scale, vector):
    dtype, d, keys = q.dtype, q.shape[-1], k.shape[1]
    if not keys:
        return TINY[dtype] + 0 * expected
    magnitude = scale * max(float((q[i].double().abs().reshape(-1, d) @ k[i].double().abs().reshape(-1, d).t()).max()) for i in range(len(q)))
    relative = 2 * ((d + 2) * U * magnitude + 5 * U * magnitude) + (3 * keys + 32) * U + 8 * (vector + 8) * U + (R.HALF[dtype] if dtype != F32 else 0.0)
    return relative * size * (1 + 2.0 ** -7) + R.HALF[dtype] * expected.abs() + TINY[dtype]


def check_attention(b, sq, sk, h, g, d, dtype, lengths=None, causal=0, scale=None, seed=0, vector=16, spread=2.0, change=None):
    q, k, v = normal(seed + 1, b, sq, 2 * h, d, scale=spread, dtype=dtype), normal(seed + 2, b, sk, 2 * g, d, dtype=dtype), normal(seed + 3, b, sk, g, 2 * d, dtype=dtype)
    vectors = [normal(seed + 4 + i, vector, scale=0.3) for i in range(4)]
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32).cuda()
    expected, size = R.differential_attention(q, k, v, vectors, 0.4, scale, n, bool(causal))
    bound = attention_bound(q, k, size, expected, scale or d ** -0.5, vector)
    if change:
        change(k, v)
    attributes = {"lambda_init": 0.4, "causal": causal, **({} if scale is None else {"scale": scale})}
    m = R.model("DifferentialAttention", [("q", q), ("k", k), ("v", v)] + [(f"l{i}", w) for i, w in enumerate(vectors)] + [("n", n)],
                [("o", dtype, (b, sq, h, 2 * d))], **attributes)
    inputs = [q, k, v, *vectors] + ([n] if n is not None else [])
    o = m(*inputs)
    assert o.dtype == dtype
    within(o, expected, bound)
    assert torch.equal(o, m(*inputs))   # whatever order workgroups run in
    return o


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("b, sq, sk, h, g", [(1, 1, 1, 1, 1), (1, 2, 3, 1, 1), (2, 31, 33, 2, 1), (1, 65, 65, 2, 2), (2, 129, 200, 3, 3), (1, 5, 700, 4, 2), (1, 200, 64, 2, 1)])
def test_attention(dtype, d, causal, b, sq, sk, h, g):
    check_attention(b, sq, sk, h, g, d, dtype, causal=causal)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("b, sq, sk, h, g", [(1, 1, 5000, 8, 2), (3, 1, 1000, 4, 4), (2, 1, 2049, 12, 2), (9, 1, 96, 40, 1), (2, 4, 3001, 4, 1)])
def test_attention_of_few_rows(dtype, d, b, sq, sk, h, g):
    lengths = [sk - 7 * i * i for i in range(b)]
    check_attention(b, sq, sk, h, g, d, dtype, lengths=lengths, causal=1)


@pytest.mark.parametrize("form", range(4))
@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("b, sq, sk, h, g", [(1, 3, 40, 2, 1), (2, 150, 129, 2, 2), (8, 130, 300, 1, 1), (1, 70, 260, 4, 1)])
def test_attention_by_every_kernel(form, dtype, d, causal, b, sq, sk, h, g, tuning):
    tuning(MI355X_DIFF_FORM=form)
    check_attention(b, sq, sk, h, g, d, dtype, causal=causal, lengths=[sk - 3 * i for i in range(b)])


@pytest.mark.parametrize("splits", [2, 5, 100])
@pytest.mark.parametrize("sq, sk", [(1, 700), (90, 333)])
def test_attention_in_any_number_of_parts(splits, sq, sk, tuning):
    for dtype in R.TYPES:
        tuning(MI355X_DIFF_SPLITS=splits)
        check_attention(2, sq, sk, 4, 2, 64, dtype, causal=1, lengths=[sk, sq + 5])


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("sq, sk", [(1, 1500), (70, 100)])
def test_attention_lengths(dtype, causal, sq, sk):
    """No key, one key, every key, more than there are and fewer than none; what lies behind a length is not a number."""
    lengths = [0, 1, sk, sk + 5, -3, 33]

    def change(k, v):
        for i, n in enumerate(lengths):
            k[i, max(n, 0):], v[i, max(n, 0):] = torch.nan, torch.inf
    o = check_attention(6, sq, sk, 4, 2, 64, dtype, lengths=lengths, causal=causal, change=change)
    assert (o[0] == 0).all() and (o[4] == 0).all()


def test_attention_without_keys_and_without_learned_vectors():
    o = check_attention(2, 3, 0, 2, 1, 64, F32)
    assert (o == 0).all()
    check_attention(1, 3, 9, 2, 1, 64, F32, vector=0)
    check_attention(1, 3, 9, 2, 1, 64, F32, vector=200)


@pytest.mark.parametrize("dtype", R.TYPES)
def test_attention_of_far_scores(dtype):
    """Scores of hundreds: the running maximum moves a long way, in either order of the keys."""
    for flip in (False, True):
        q, k, v = normal(1, 1, 40, 4, 64, scale=20, dtype=dtype), normal(2, 1, 300, 2, 64, scale=2, dtype=dtype), normal(3, 1, 300, 1, 128, dtype=dtype)
        k = (k.float() * torch.linspace(0.01, 2, 300).cuda().flip(0 if flip else ())[None, :, None, None]).to(dtype)
        vectors = [normal(4 + i, 8, scale=0.3) for i in range(4)]
        expected, size = R.differential_attention(q, k, v, vectors, 0.4)
        o, = R.call("DifferentialAttention", [("q", q), ("k", k), ("v", v)] + [(f"l{i}", w) for i, w in enumerate(vectors)], [("o", dtype, (1, 40, 2, 128))], lambda_init=0.4)
        within(o, expected, attention_bound(q, k, size, expected, 0.125, 8))


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("sq", [1, 40])
@pytest.mark.parametrize("first", [0, 777, 19999])
def test_attention_of_many_keys_of_little_weight(dtype, sq, first):
    """One key has nearly all of the weight and no value, 19999 others share 2^-9 of it. (Scores are exact, 0 and 16.)"""
    b, sk, h, d = 1, 20000, 2, 64
    q, k, v = normal(1, b, sq, 2 * h, d, dtype=dtype), torch.zeros(b, sk, 2, d, dtype=dtype, device="cuda"), normal(3, b, sk, 1, 2 * d, dtype=dtype).abs()
    q[..., 0] = 2.0 ** 4
    k[:, first, :, 0], v[:, first] = 1.0, 0.0
    vectors = [normal(4 + i, 8, scale=0.3) for i in range(4)]
    expected, size = R.differential_attention(q, k, v, vectors, 0.4, 1.0)
    o, = R.call("DifferentialAttention", [("q", q), ("k", k), ("v", v)] + [(f"l{i}", w) for i, w in enumerate(vectors)], [("o", dtype, (b, sq, h, 2 * d))], lambda_init=0.4, scale=1.0)
    within(o, expected, attention_bound(q, k, size, expected, 1.0, 8))


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("sq, splits", [(5, 1), (5, 3), (1, 7), (5, 256)])
def test_attention_at_any_address_and_any_splits(dtype, sq, splits):
    lib, (b, sk, h, g, d) = _lib.library(), (2, 150, 4, 2, 64)
    shapes = [(b, sq, 2 * h, d), (b, sk, 2 * g, d), (b, sk, g, 2 * d), (b, sq, h, 2 * d)]
    buffers = [torch.zeros(math.prod(s) + 9, dtype=dtype, device="cuda") for s in shapes]
    q, k, v, o = (t[i + 1:i + 1 + math.prod(s)].view(s) for i, (t, s) in enumerate(zip(buffers, shapes)))
    for i, t in enumerate((q, k, v)):
        t.copy_(normal(i, *t.shape, dtype=dtype))
    vectors = [normal(4 + i, 8, scale=0.3) for i in range(4)]
    scratch = torch.full((splits * b * sq * h * (4 * d + 4) + 64,), 7.0, device="cuda")
    _lib.check(lib.mi355x_differential_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), *(w.data_ptr() for w in vectors), None, o.data_ptr(), scratch.data_ptr(), b, sq, sk, h, g, d, 8,
                                                 0.4, 0.125, 1, splits, R.ELEMENT[dtype], _lib.current_stream()), "attention")
    expected, size = R.differential_attention(q, k, v, vectors, 0.4, 0.125, None, True)
    within(o, expected, attention_bound(q, k, size, expected, 0.125, 8))
    assert (scratch[-64:] == 7).all() and buffers[3][:4].abs().max() == 0 and buffers[3][4 + o.numel():].abs().max() == 0


def test_attention_of_a_cache_beyond_32_bits():
    """2^31 values and more to keys and values each; the last keys weigh most."""
    b, sk, g, d = 1, 1100000, 8, 128
    k = torch.zeros(b, sk, 2 * g, d, dtype=BF, device="cuda")
    v = torch.zeros(b, sk, g, 2 * d, dtype=BF, device="cuda")
    assert k.numel() > 1 << 31
    q = normal(1, b, 1, 2 * g, d, dtype=BF)
    places = torch.tensor([0, 1, 70000, 1048577, sk - 33, sk - 1]).cuda()
    k[:, places], v[:, places] = normal(2, b, 6, 2 * g, d, scale=3, dtype=BF), normal(3, b, 6, g, 2 * d, scale=1000, dtype=BF)
    vectors = [normal(4 + i, 8, scale=0.3) for i in range(4)]
    o, = R.call("DifferentialAttention", [("q", q), ("k", k), ("v", v)] + [(f"l{i}", w) for i, w in enumerate(vectors)], [("o", BF, (b, 1, g, 2 * d))], lambda_init=0.4, scale=1.0)
    # the other keys have a score of 0 and no value: they only count
    few, many = places.numel(), sk - places.numel()
    weight = math.exp(float(vectors[0].double() @ vectors[1].double())) - math.exp(float(vectors[2].double() @ vectors[3].double())) + 0.4
    s = torch.einsum("hmd,nhmd->hmn", q[0, 0].double().view(g, 2, d), k[0, places].double().view(few, g, 2, d))
    top = s.amax(-1, keepdim=True).clamp(min=0)
    p = torch.exp(s - top) / (torch.exp(s - top).sum(-1, keepdim=True) + many * torch.exp(-top))
    value = v[0, places].double().transpose(0, 1)   # [g, few, 2 d]
    expected = ((p[:, 0] - weight * p[:, 1])[:, None] @ value)[:, 0]
    size = ((p[:, 0] + abs(weight) * p[:, 1])[:, None] @ value.abs())[:, 0]
    # the scores reach sum |q k|; a sum over the keys that a workgroup and a lane adds up, and over the splits, counts as in the bound above
    magnitude = float((q[0, 0].double().abs().view(g, 2, 1, d) * k[0, places].double().abs().view(few, g, 2, d).permute(1, 2, 0, 3)).sum(-1).max())
    relative = 2 * (d + 7) * U * magnitude + (3 * sk / 16 + 32) * U + 8 * 16 * U + R.HALF[BF]
    within(o[0, 0], expected, relative * size + R.HALF[BF] * expected.abs())


# ---------------------------------------------------------------------------------------------- together


def layer(rng, batch, seq, cache, hidden, heads, groups, d, dtype):
    """One layer of a differential transformer with quantised projections over a cache, as nodes of a graph and as its weights."""
    T = R.ELEMENT[dtype]
    weights, nodes = {}, []

    def weight(name, value, kind=None):
        weights[name] = helper.make_tensor(name, T, value.shape, value) if kind is None else numpy_helper.from_array(value.astype(kind), name)
        return name

    def linear(x, scale, rows, name, residual="", activation="none"):
        weight(name, rng.integers(-127, 128, (rows, hidden)), np.int8), weight(name + "_scale", rng.uniform(0.5, 1, rows) / 74 / hidden ** 0.5, np.float32)
        weight(name + "_bias", rng.normal(size=rows) * 0.1)
        nodes.append(helper.make_node("QuantizedLinear", [x, name, scale, name + "_scale", name + "_bias", residual], [name + "_y"], name=name, activation=activation, to=T))
        return name + "_y"

    weight("gain", 1 + 0.1 * rng.normal(size=hidden)), weight("head_gain", 0.5 + 0.1 * rng.normal(size=2 * d)), weight("gain2", 1 + 0.1 * rng.normal(size=hidden))
    weight("frequencies", 100.0 ** (-np.arange(d // 2) / (d // 2)), np.float32)
    for n in ("q1", "k1", "q2", "k2"):
        weight("lambda_" + n, rng.normal(size=d) * 0.1, np.float32)
    nodes.append(helper.make_node("SkipRMSNormalization", ["x", "gain", "skip"], ["", "stream", "x8", "x8_scale"], name="norm"))
    shaped = {"q": (linear("x8", "x8_scale", 2 * heads * d, "wq"), [batch, seq, 2 * heads, d]), "k": (linear("x8", "x8_scale", 2 * groups * d, "wk"), [batch, seq, 2 * groups, d]),
              "v": (linear("x8", "x8_scale", 2 * groups * d, "wv"), [batch, seq, groups, 2 * d])}
    for name, (y, shape) in shaped.items():
        nodes.append(helper.make_node("Reshape", [y, weight(name + "_shape", np.array(shape), np.int64)], [name], name="split_" + name))
    nodes.append(helper.make_node("RotaryPositions", ["q", "positions", "frequencies", "k"], ["q_turned", "k_turned"], name="rotary", sections=[d // 2 - 2 * (d // 6), d // 6, d // 6]))
    nodes.append(helper.make_node("DifferentialAttention", ["q_turned", "k_turned", "v"] + ["lambda_" + n for n in ("q1", "k1", "q2", "k2")] + ["lengths"], ["o"], name="attention",
                                  causal=1, lambda_init=0.3))
    nodes.append(helper.make_node("SkipRMSNormalization", ["o", "head_gain"], ["o_normed"], name="head_norm"))
    nodes.append(helper.make_node("Reshape", ["o_normed", weight("merged", np.array([batch, seq, hidden]), np.int64)], ["merged_o"], name="merge"))
    nodes.append(helper.make_node("SkipRMSNormalization", ["merged_o", "gain2"], ["", "", "o8", "o8_scale"], name="norm2"))
    out = linear("o8", "o8_scale", hidden, "wo", residual="stream", activation="silu")
    inputs = [("x", T, (batch, seq, hidden)), ("skip", T, (batch, seq, hidden)), ("positions", 7, (3, batch, seq)), ("lengths", 6, (batch,))]
    graph = helper.make_graph(nodes, "layer", [helper.make_tensor_value_info(*i[:2], list(i[2])) for i in inputs],
                              [helper.make_tensor_value_info(n, T, [batch, seq, hidden]) for n in (out, "stream")], initializer=list(weights.values()))
    return helper.make_model(graph), weights


def layer_in_float64(weights, x, skip, positions, lengths, heads, groups, d):
    """The layer step by step, each rounded as the framework's arrays between the nodes are."""
    dtype, (batch, seq, hidden) = x.dtype, x.shape
    w = {n: torch.from_numpy(np.ascontiguousarray(t.array)).cuda() for n, t in weights.items()}
    low = lambda t: t.to(dtype)  # noqa: E731

    def quantised(t, gain, skip=None):
        _, s, q, scale = R.rms_norm(t, w[gain].to(dtype), skip)
        return low(s), q.reshape(-1, hidden), scale.reshape(-1)

    def linear(q, scale, name, residual=None, activation="none"):
        return low(R.quantized_linear(q, w[name], scale, w[name + "_scale"], w[name + "_bias"].to(dtype), residual, activation)[0])

    stream, q8, scale = quantised(x, "gain", skip)
    q, k, v = (linear(q8, scale, n).reshape(batch, seq, -1, c) for n, c in (("wq", d), ("wk", d), ("wv", 2 * d)))
    sections = [d // 2 - 2 * (d // 6), d // 6, d // 6]
    q, k = (low(R.rotary(t, positions, w["frequencies"], sections, False)) for t in (q, k))
    o = low(R.differential_attention(q, k, v, [w["lambda_" + n] for n in ("q1", "k1", "q2", "k2")], 0.3, None, lengths, True)[0])
    o = low(R.rms_norm(o, w["head_gain"].to(dtype))[0]).reshape(batch, seq, hidden)
    _, o8, o_scale = quantised(o, "gain2")
    return linear(o8, o_scale, "wo", stream.reshape(-1, hidden), "silu").reshape(batch, seq, hidden), stream


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("batch, seq, heads, groups, d", [(2, 45, 4, 2, 32), (3, 1, 2, 1, 64), (1, 150, 2, 2, 128)])
def test_a_layer(dtype, batch, seq, heads, groups, d):
    hidden = 2 * heads * d
    model, weights = layer(np.random.default_rng(3), batch, seq, seq, hidden, heads, groups, d, dtype)
    x, skip = normal(1, batch, seq, hidden, dtype=dtype), normal(2, batch, seq, hidden, dtype=dtype)
    positions = torch.randint(0, 1000, (3, batch, seq), generator=torch.Generator().manual_seed(4)).cuda()
    lengths = torch.tensor([seq] * batch, dtype=torch.int32).cuda()
    expected, stream = layer_in_float64(weights, x, skip, positions, lengths, heads, groups, d)
    m = donnx.ONNXModel("layer", model)
    out, got_stream = m(x, skip, positions, lengths)
    assert out.dtype == dtype and torch.equal(got_stream, stream)
    # Values are rounded to eight bits twice on the way. A value at a border that goes the other way is a step of eight bits off, 2 / 127 of its row's largest half,
    # and few do: per step of the 16-bit arrays between the nodes (of float32 there is none to speak of) fewer than one in ten of the others. In the 2-norm:
    # (1 / 127) sqrt(1 / 10) for each of the two, and three steps of the arrays' type.
    bound = 2 / 127 * 0.1 ** 0.5 + 3 * 2 * R.HALF[dtype]
    assert float((out.double() - expected.double()).norm() / expected.double().norm()) < bound
    replayed = donnx.ONNXModel("layer", model, use_hip_graph=True)
    for _ in range(4):   # recorded, then replayed with eager work between
        assert torch.equal(replayed(x, skip, positions, lengths)[0], out)
        assert torch.equal(m(x, skip, positions, lengths)[0], out)
        torch.cuda.synchronize()


def test_a_layer_from_numpy():
    model, weights = layer(np.random.default_rng(3), 1, 5, 5, 128, 2, 1, 32, BF)
    x, skip = normal(1, 1, 5, 128, dtype=BF), normal(2, 1, 5, 128, dtype=BF)
    positions, lengths = torch.arange(15).reshape(3, 1, 5), torch.tensor([5], dtype=torch.int32)
    m = donnx.ONNXModel("layer", model)
    expected = m(x, skip, positions.cuda(), lengths.cuda())
    got = m(x.float().cpu().numpy(), skip.float().cpu().numpy(), positions.numpy(), lengths.numpy())
    assert all(isinstance(a, np.ndarray) and a.dtype == np.float32 and np.array_equal(a, b.float().cpu().numpy()) for a, b in zip(got, expected))


def test_calls_of_single_nodes_write_into_the_callers_tensors():
    x, gain = normal(1, 6, 64, dtype=BF), normal(2, 64, dtype=BF)
    y, q, scale = torch.empty_like(x), torch.empty(6, 64, dtype=torch.int8, device="cuda"), torch.empty(6, device="cuda")
    donnx.ONNXSkipRMSNormalization(X=x, Scale=gain, Y=y, Q=q, q_scale=scale)
    check_norm(x, gain, None, y, None, q, scale)
    w, out = eight(3, 32, 64), torch.empty(6, 32, device="cuda")
    donnx.ONNXQuantizedLinear(X=q, W=w, x_scale=scale, w_scale=torch.ones(1, device="cuda"), Y=out)
    expected, size = R.quantized_linear(q, w, scale, torch.ones(32, device="cuda"))
    within(out, expected, linear_bound(size, expected, F32))
    with pytest.raises(donnx.ExpansionRefused):
        donnx.ONNXQuantizedLinear(X=q, W=w, x_scale=scale, w_scale=torch.ones(3, device="cuda"), Y=out)


def test_another_stream_and_recordings_of_the_caller():
    """Calls on a side stream, and captured by the caller: replays follow inputs that are written between them."""
    q, k, v = normal(1, 2, 1, 8, 64, dtype=BF), normal(2, 2, 4000, 4, 64, dtype=BF), normal(3, 2, 4000, 2, 128, dtype=BF)
    vectors, lengths = [normal(4 + i, 8, scale=0.3) for i in range(4)], torch.tensor([4000, 17], dtype=torch.int32).cuda()
    inputs = [("q", q), ("k", k), ("v", v)] + [(f"l{i}", w) for i, w in enumerate(vectors)] + [("n", lengths)]
    m = R.model("DifferentialAttention", inputs, [("o", BF, (2, 1, 4, 128))], causal=1)
    tensors = [t for _, t in inputs]
    first = m(*tensors)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(m(*tensors), first)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m(*tensors)
    for n in ((4000, 17), (1, 0), (2000, 4000), (33, 64)):
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        assert torch.equal(replayed, m(*tensors))
        torch.cuda.synchronize()


def test_attention_in_parts_as_a_recorded_graph_and_as_a_single_call():
    """A graph that has the sums of its parts recorded with it, replayed between eager calls; a node called by itself on two streams in turn."""
    q, k, v = normal(1, 2, 1, 8, 64, dtype=F16), normal(2, 2, 3000, 4, 64, dtype=F16), normal(3, 2, 3000, 2, 128, dtype=F16)
    vectors, lengths = [normal(4 + i, 8, scale=0.3) for i in range(4)], torch.tensor([3000, 17], dtype=torch.int32).cuda()
    assert _lib.library().mi355x_differential_attention_splits(2, 1, 3000, 4, 2, 64, 10) > 1
    names = ["Q", "K", "V", "lambda_q1", "lambda_k1", "lambda_q2", "lambda_k2", "lengths"]
    tensors = [q, k, v, *vectors, lengths]
    infos = [helper.make_tensor_value_info(n, R.ELEMENT[t.dtype], list(t.shape)) for n, t in zip(names, tensors)]
    graph = helper.make_model(helper.make_graph([helper.make_node("DifferentialAttention", names, ["O"], name="node", causal=1, lambda_init=0.4)], "one", infos,
                                                [helper.make_tensor_value_info("O", 10, [2, 1, 4, 128])]))
    eager, recorded = donnx.ONNXModel("eager", graph), donnx.ONNXModel("recorded", graph, use_hip_graph=True)
    out, side = torch.empty(2, 1, 4, 128, dtype=F16, device="cuda"), torch.cuda.Stream()
    for n in ((3000, 17), (1, 0), (2000, 3000), (33, 64)):
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        expected, size = R.differential_attention(q, k, v, vectors, 0.4, None, lengths, True)
        o = eager(*tensors).clone()
        within(o, expected, attention_bound(q, k, size, expected, 0.125, 8))
        assert torch.equal(recorded(*tensors), o)
        for stream in (torch.cuda.current_stream(), side):
            stream.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(stream):
                donnx.ONNXDifferentialAttention(**dict(zip(names, tensors)), O=out, causal=1, lambda_init=0.4)
            torch.cuda.default_stream().wait_stream(stream)
            assert torch.equal(out, o)
            out.zero_()


@pytest.mark.parametrize("form", range(5))
@pytest.mark.parametrize("m, n, k", [(512, 512, 64), (300, 270, 144), (257, 515, 33)])
@pytest.mark.parametrize("residual", [False, True])
def test_linear_results_of_a_tile_are_where_they_belong(form, m, n, k, residual, tuning):
    """Whole numbers, equal to the last bit: no row of a tile has another's results, whichever lanes hand them round."""
    tuning(MI355X_QLIN_FORM=form)
    x, w, one = eight(1, m, k), eight(2, n, k), torch.ones(1, device="cuda")
    r = eight(3, m, n).float() if residual else None
    expected = (x.double() @ w.double().t() + (r.double() if residual else 0)).float()
    for _ in range(3):
        y, = R.call("QuantizedLinear", [("x", x), ("w", w), ("xs", one), ("ws", one), ("b", None), ("r", r)], [("y", F32, (m, n))])
        assert torch.equal(y, expected)


@pytest.mark.parametrize("dtype, d", [(BF, 128), (F16, 128), (F32, 64)])
@pytest.mark.parametrize("causal", [0, 1])
def test_attention_of_many_rows_of_wide_heads_in_parts(dtype, d, causal):
    """Heads of 256 bytes with more than 128 blocks of 32 rows: two row waves and two key waves to a workgroup, and the keys in parts."""
    assert _lib.library().mi355x_differential_attention_splits(2, 2100, 2200, 1, 1, d, R.ELEMENT[dtype]) > 1
    check_attention(2, 2100, 2200, 1, 1, d, dtype, causal=causal, lengths=[2200, 2101])
