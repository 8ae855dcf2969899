"""The rest of a decoder's step on the GPU at the ends of its ranges: values with all their bits, few pairs among many
experts.  Tolerances count roundings, each half a step (2^-24 of a value in fp32, 2^-8 in bf16), or are those of
tests/test_gpu_decoder_step.py."""
from __future__ import annotations

import numpy as np
import pytest

import oracle
from oracle import decoder_step as od
from oct_amd import prometheus as p
from tests.test_gpu_decoder_step import BF16, F32, HALF_STEP, _close, _matrix, _mixture, _product
from tests.test_gpu_quantised_path import Device, _bits, _rounded, _values

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


# ------------------------------------------------------------------ the mixture's hidden rows
def _held(shape, at):
    """Weights that groups of 32 hold exactly: `at` gives {(row, column): power of two}; the column behind each is six
    times as large, so that the step is that power (and has to meet a zero)."""
    w = np.zeros(shape, np.float32)
    for (row, column), value in at.items():
        w[row, column], w[row, column + 1] = value, 6.0 * abs(value)
    return w


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("tokens", (1, 12, 40, 130))
def test_hidden_rows_keep_all_their_bits(gpu_runtime, tokens, dtype):
    """out = h1 - h2 for two hidden values of 24 bits that differ in the last eight: 32 (x0 + x32 / 2^8 + x64 / 2^16) and
    the same without its last summand, from bf16 numbers in [1, 2).  The gate is 32, whose activation is 32 to 2^-46.
    Every sum is exact but for a few roundings of what is left."""
    hidden, inner = 128, 70
    x = np.zeros((tokens, hidden), np.float32)
    x[:, [0, 32, 64]] = _rounded(oracle.uniform(tokens, (tokens, 3), 1.0, 2.0), BF16)
    x[:, 96] = 32.0
    gate = np.zeros((inner, hidden), np.float32)
    gate[[3, 40]] = _held((1, hidden), {(0, 96): 1.0})
    up = np.zeros((inner, hidden), np.float32)
    up[3] = _held((1, hidden), {(0, 0): 1.0, (0, 32): 2.0 ** -8, (0, 64): 2.0 ** -16})
    up[40] = _held((1, hidden), {(0, 0): 1.0, (0, 32): 2.0 ** -8})
    scales = np.exp2(np.arange(hidden) % 5).astype(np.float32)
    down = np.zeros((hidden, inner), np.float32)
    down[:, 3], down[:, 4], down[:, 40], down[:, 41] = scales, 6 * scales, -scales, 6 * scales
    router = np.ones((1, hidden), np.float32)
    with Device(gpu_runtime) as dev:
        (gate, gv), (up, uv), (down, dv) = (_matrix(dev, w[None], 32) for w in (gate, up, down))
        assert gv.max() == 6 and uv[0, 3, 64] == 2.0 ** -16 and np.array_equal(dv[0, :, 3], scales)
        out = _bits(np.zeros((tokens, hidden), np.float32), dtype)
        to = dev.up(out)
        gpu_runtime.moe_w4_device(gate, up, down, dev.up(router), dev.up(_bits(x, dtype)), to, tokens, 1, hidden, hidden, dtype)
        got = _values(dev.down(out, to), dtype).astype(np.float64)
    expect = 32.0 * 2.0 ** -16 * x[:, 64:65].astype(np.float64) * scales
    # activation and hidden values to 2^-46; two sums of terms that cancel exactly but for their last eight bits
    assert np.all(np.abs(got - expect) <= (HALF_STEP[dtype] + 4 * U) * expect)


# ------------------------------------------------------------------ few pairs among many experts
@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("tokens,experts,top_k,group,renormalise", [
    (65, 131, 1, 32, False), (65, 132, 1, 64, True), (100, 256, 1, 32, True), (128, 1024, 2, 128, False),
    (128, 1024, 3, 64, True), (70, 300, 2, 32, False)])
def test_mixture_of_fewer_pairs_than_half_the_experts(gpu_runtime, tokens, experts, top_k, group, renormalise, dtype):
    case = dict(tokens=tokens, hidden=64, inner=48, experts=experts, top_k=top_k, group=group, renormalise=renormalise)
    _close(*_mixture(gpu_runtime, case, dtype), dtype)


# ------------------------------------------------------------------ products of fp32 rows with all their bits
def _single(rows, k, low, high, seed=3):
    """Rows with one number each, of 24 significant bits, at columns that meet every part of a K tile."""
    x = np.zeros((rows, k), np.float32)
    columns = (np.arange(rows) * 53 + k - 1) % k
    bits = np.random.default_rng(seed).integers(1 << 23, 1 << 24, rows).astype(np.float64)
    x[np.arange(rows), columns] = np.ldexp(bits, np.random.default_rng(seed + 1).integers(low, high, rows) - 23)
    x[::3] *= -1
    return x, columns


@pytest.mark.parametrize("group", (32, 64, 128))
@pytest.mark.parametrize("rows,n,k", [(3, 47, 395), (16, 600, 256), (20, 40, 9001), (40, 4500, 131), (5, 40, 6),
                                      (200, 47, 395), (300, 260, 256), (1024, 4000, 256), (1000, 4000, 395), (1024, 4000, 7),
                                      (512, 2000, 1000)])  # the last four on tiles
def test_fp32_rows_enter_with_all_their_bits(gpu_runtime, rows, n, k, group):
    """x w from three terms.  The sums of the last two are exact to 2^-8 of a rounding; that with the first is within 2^-23,
    as a matrix instruction may cut it off, and the product with the step within half of that.  Zeros' sums are exact."""
    x, columns = _single(rows, k, -6, 7)
    w = (oracle.normal(n, (n, k)) * np.exp2(oracle.uniform(2, (n, 1), -3.0, 3.0))).astype(np.float32)
    got, values = _product(gpu_runtime, x, w, group, F32)
    expect = x[np.arange(rows), columns].astype(np.float64)[:, None] * values[:, columns].T
    assert np.all(np.abs(got - expect) <= 3.1 * U * np.abs(expect))


@pytest.mark.parametrize("group", (32, 64, 128))
@pytest.mark.parametrize("n", (100, 2400, 4800, 13600, 32800))
@pytest.mark.parametrize("k", (7, 131, 256))
def test_every_column_of_fp32_rows_enters_with_all_its_bits(gpu_runtime, n, k, group):
    """As above, for each column of a K tile and of its rest, with one to eight waves a workgroup and 32 or 64 columns."""
    w = (oracle.normal(n, (n, k)) * np.exp2(oracle.uniform(2, (n, 1), -3.0, 3.0))).astype(np.float32)
    with Device(gpu_runtime) as dev:
        matrix, values = _matrix(dev, w, group)
        out = np.zeros((64, n), np.float32)
        to = dev.up(out)
        for first in range(0, k, 64):
            columns = (first + np.arange(64)) % k
            x = np.zeros((64, k), np.float32)
            x[np.arange(64), columns] = np.random.default_rng(first).integers(1 << 23, 1 << 24, 64) * np.float32(2.0 ** -23)
            gpu_runtime.gemm_w4_device(matrix, dev.up(x), to, 64, k, n, F32)
            expect = x[np.arange(64), columns].astype(np.float64)[:, None] * values[:, columns].T
            assert np.all(np.abs(dev.down(out, to) - expect) <= 3.1 * U * np.abs(expect)), first


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("rows,n", ((20, 40), (1024, 4000)))
def test_products_with_the_largest_weights(gpu_runtime, rows, n, dtype):
    """Weights up to the largest that stay finite, exactly, in both kernels; zeros beside them stay zeros."""
    k, most = 256, 63 * 2.0 ** 122
    w = np.clip(oracle.normal(n, (n, k)).astype(np.float64) * 2.0 ** 127, -most, most).astype(np.float32)
    columns = (np.arange(rows) * 53) % k
    x = np.zeros((rows, k), np.float32)
    x[np.arange(rows), columns] = np.exp2(-(np.arange(rows) % 9))
    got, values = _product(gpu_runtime, x, w, 64, dtype)
    assert np.array_equal(got, x[np.arange(rows), columns].astype(np.float64)[:, None] * values[:, columns].T)


@pytest.mark.parametrize("group", (32, 64, 128))
@pytest.mark.parametrize("hidden", (256, 260))
@pytest.mark.parametrize("tokens,experts", ((64, 1), (255, 1), (64, 64), (255, 64)))
def test_every_column_of_a_mixture_enters_with_all_its_bits(gpu_runtime, tokens, experts, hidden, group):
    """A token has one number x besides its gate's, which makes one hidden value h = 48 (6 x), and out = h down[:, f]: x
    and h are 24 bits each.  The sum 6 x and the last one are within 3.1 halves of a step, h, its activation, the weight 1
    and the sum over experts are a rounding each."""
    inner = 250
    up = np.zeros((inner, hidden), np.float32)
    up[np.arange(inner), np.arange(inner)] = 6.0
    gate = np.zeros((inner, hidden), np.float32)
    gate[:, hidden - 1] = 6.0
    down = oracle.normal(4, (hidden, inner))
    router = oracle.normal(5, (experts, hidden))
    with Device(gpu_runtime) as dev:
        matrices, values = [], None
        for w in (gate, up, down):
            codes, steps = od.w4_quantise(w, group)
            values = od.w4_values(codes, steps, group)
            matrices.append(p.w4_matrix(dev.up(np.tile(od.w4_pack(codes, steps, group), experts)), *w.shape, group, experts))
        assert np.array_equal(od.w4_values(*od.w4_quantise(up, group), group), up)
        out, drouter = np.zeros((tokens, hidden), np.float32), dev.up(router)
        to = dev.up(out)
        for first in range(0, inner, tokens):
            f = (first + np.arange(tokens)) % inner
            x = np.zeros((tokens, hidden), np.float32)
            number = np.random.default_rng(first).integers(1 << 23, 1 << 24, tokens) * np.float32(2.0 ** -23)
            x[np.arange(tokens), f], x[:, -1] = number, 8.0
            gpu_runtime.moe_w4_device(*matrices, drouter, dev.up(x), to, tokens, 1, hidden, hidden, F32, renormalise=True)
            expect = 288.0 * number.astype(np.float64)[:, None] * values[:, f].T
            assert np.all(np.abs(dev.down(out, to) - expect) <= 11 * U * np.abs(expect)), first


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("rows,n", ((20, 40), (1000, 4000)))
def test_products_of_the_smallest_rows(gpu_runtime, rows, n, dtype):
    """Elements down to fp32's smallest: what a term of eight bits holds ends at 2^-133, bf16's smallest number, so that
    fp32 elements are exact down to 2^-110 and within 2^-133 below."""
    k = 300
    x, columns = _single(rows, k, -126, -100)
    x = _rounded(x, dtype)
    w = (oracle.normal(n, (n, k)) * 2.0 ** 60).astype(np.float32)
    got, values = _product(gpu_runtime, x, w, 64, dtype)
    expect = x[np.arange(rows), columns].astype(np.float64)[:, None] * values[:, columns].T
    left_out = np.abs(values[:, columns].T) * (2.0 ** -133 if dtype == F32 else 0.0)
    assert np.all(np.abs(got - expect) <= left_out + (3.1 * U + (HALF_STEP[BF16] if dtype == BF16 else 0.0)) * np.abs(expect))


# ------------------------------------------------------------------ logits without a value
@pytest.mark.parametrize("renormalise", (False, True))
@pytest.mark.parametrize("experts,tokens", ((6, 1), (6, 20), (70, 3), (300, 170)))
def test_weights_are_nan_where_a_logit_is(gpu_runtime, experts, tokens, renormalise):
    """A softmax over all experts has no value where one of its logits has none, chosen or not: the choice goes by the
    others, the weights and the row of that token are NaN.  The other tokens' logit of that expert is below all numbers."""
    hidden, inner, top_k = 64, 32, 2
    x = oracle.normal(3, (tokens, hidden))
    x[:, 5] = -1.0
    x[0, 5] = 0.0
    router = (oracle.normal(5, (experts, hidden)) * 0.2).astype(np.float32)
    router[2, 5] = np.inf
    shapes = ((inner, hidden), (inner, hidden), (hidden, inner))
    with Device(gpu_runtime) as dev:
        matrices = [_matrix(dev, oracle.normal(i, (experts, *shape)) * np.float32(0.1), 32)[0] for i, shape in enumerate(shapes)]
        out, chosen = np.zeros((tokens, hidden), np.float32), np.zeros((tokens, top_k), np.int32)
        weights = np.zeros((tokens, top_k), np.float32)
        to, dc, dw = dev.up(out), dev.up(chosen), dev.up(weights)
        gpu_runtime.moe_w4_device(*matrices, dev.up(router), dev.up(x), to, tokens, top_k, hidden, hidden, F32,
                                  renormalise=renormalise, dexperts=dc, dweights=dw)
        out, chosen, weights = dev.down(out, to), dev.down(chosen, dc), dev.down(weights, dw)
    with np.errstate(invalid="ignore"):
        expect_chosen, expect = od.route(x, router, top_k, renormalise)
    assert np.array_equal(chosen, expect_chosen) and not (chosen == 2).any()
    assert np.isnan(weights[0]).all() and np.isnan(out[0]).all() and np.isfinite(out[1:]).all()
    assert np.allclose(weights, expect, rtol=2.0 ** -22, equal_nan=True)


# ------------------------------------------------------------------ rotary positions
@pytest.mark.parametrize("pairs", (False, True))
@pytest.mark.parametrize("magnitude", (1.0, 1.2079441541679836))
@pytest.mark.parametrize("rows", (300, 4100))
def test_rope_rounds_only_at_its_end(gpu_runtime, rows, magnitude, pairs):
    """Angle, cosine, sine and magnitude in binary64, the last three's product rounded once to fp32, then a product, a fused
    one and no other rounding: 2 |a c| + 3 |b s| halves of a step at most, in either order.  Such errors, spread evenly over
    a step, have a mean square of at most a third of (a c)^2 + 2 (b s)^2 + out^2 halves of a step: 5/6 of x^2 over all."""
    heads, dim = 2, 64
    positions = np.random.default_rng(rows).integers(0, 1 << 20, rows).astype(np.int32)
    turns, _ = p.rope_turns(dim)
    x = _rounded(oracle.normal(rows, (rows, heads * dim)), F32)
    with Device(gpu_runtime) as dev:
        to = dev.up(x)
        gpu_runtime.rope_device(dev.up(positions), dev.up(turns), rows, dim, dim, p.ROPE_PAIRS if pairs else p.ROPE_HALF, F32,
                                magnitude, q=(to, to, heads, heads * dim, heads * dim))
        got = dev.down(x, to).reshape(rows, heads, dim).astype(np.float64)
    magnitude = float(np.float32(magnitude))
    x = x.reshape(rows, heads, dim).astype(np.float64)
    t = positions.astype(np.longdouble)[:, None] * turns.astype(np.longdouble)
    angle = 2.0 * np.pi * (t - np.rint(t)).astype(np.float64)
    c, s = (magnitude * f(angle)[:, None] for f in (np.cos, np.sin))
    # positions * turns is rounded to 2^-53 of itself, 2^20 / (2 pi) at most: 2^-35 of a turn, far below U
    off = 2 * np.pi * np.abs(t).astype(np.float64)[:, None] * 2.0 ** -53 * magnitude + magnitude * 2.0 ** -40
    first = np.arange(dim // 2) * 2 if pairs else np.arange(dim // 2)
    second = first + 1 if pairs else first + dim // 2
    a, b = x[..., first], x[..., second]
    square = 0.0
    for out, u, v, f, g in ((first, a, b, c, -s), (second, b, a, c, s)):
        expect = u * f + v * g
        limit = U * (3 * np.abs(u * f) + 3 * np.abs(v * g)) * (1 + 2.0 ** -20) + (np.abs(u) + np.abs(v)) * off
        assert np.all(np.abs(got[..., out] - expect) <= limit)
        square += ((got[..., out] - expect) ** 2).sum()
    assert square <= 5.0 / 6.0 * U ** 2 * magnitude ** 2 * (x * x).sum()


# ------------------------------------------------------------------ residual norms
@pytest.mark.parametrize("width", (8, 601, 1504, 16400))
def test_residual_norm_at_the_ends_of_the_range(gpu_runtime, width):
    """Rows of the smallest and largest numbers: 1 / sqrt of the mean may lie past fp32's range or among its subnormal
    numbers, the quotient does not.  x / size: its scaling is exact, then a factor and a product: two roundings, and one
    of the size."""
    scales = [2.0 ** -146, 2.0 ** -140, 2.0 ** -129, 2.0 ** -127, 2.0 ** -126, 2.0 ** 120, 2.0 ** 126, 1.0]
    x = np.clip(oracle.normal(1, (len(scales), width)), -1.9, 1.9).astype(np.float64)
    x = (x * np.array(scales)[:, None]).astype(np.float32)
    x[0, :2] = np.float32(2.0 ** -146)  # the smallest rows are not zeros
    weight = (oracle.normal(2, (width,)) * 0.1 + 1.0).astype(np.float32)
    h = np.zeros_like(x)
    with Device(gpu_runtime) as dev:
        dx, dw = dev.up(x), dev.up(weight)
        norm, h_out = dev.up(x), dev.up(x)
        gpu_runtime.residual_norm_device(dx, None, norm, len(x), width, F32, dpre=dw, eps=0.0)
        gpu_runtime.residual_norm_device(dev.up(h), h_out, None, len(x), width, F32, dy=dx, dpost=dw, eps=0.0)
        got = [dev.down(x, norm), dev.down(x, h_out)]
    wide = x.astype(np.float64)
    expect = wide / np.sqrt((wide ** 2).mean(1, keepdims=True)) * weight.astype(np.float64)
    for v in got:
        assert np.all(np.abs(v - expect) <= 4 * U * np.abs(expect) + 2.0 ** -140)
