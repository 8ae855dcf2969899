"""The rest of a decoder's step on the GPU against its definitions in 64 bits (oracle/decoder_step.py).

Packed matrices and what is unpacked are compared byte for byte, chosen experts exactly.  Tolerances:

product: terms are exact and sums fp32.  A matrix instruction adds 32 products to its sum in at most 33 roundings, each
within 2^-23 of what is added (whatever its order); a group of up to 128 takes 4 of them a term of x (3 terms in fp32),
which errs by at most 33 * 4 * terms * 2^-23 of the group's sum of magnitudes.  The groups' sums (times a step, one
rounding) are added in a lane, over at most 16 waves and 64 slices: K / group + 80 more roundings of 2^-24.  In units
of 2^-23 that is `_chain`.  A bf16 result is rounded once more, 2^-8 of it.

mixture: the same for each product, through the activation's slope and the second product (oracle/decoder_step.py);
hidden values enter with 16 bits (bf16 rows: 2^-17 and a rounding) or 24.  Weights are binary64 rounded to fp32 with an
exponential good to 2^-50: 2^-23 of them.

rope, residual_norm: the bounds that oracle/decoder_step.py derives, and a bf16 result's rounding."""
from __future__ import annotations

import threading

import numpy as np
import pytest

import oracle
from oracle import decoder_step as od
from oracle import quantised as oq
from oct_amd import prometheus as p
from tests.test_gpu_quantised_path import Device, _bits, _rounded, _values

pytestmark = pytest.mark.gpu

F32, BF16 = p.DTYPE_F32, p.DTYPE_BF16
HALF_STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8}


def _chain(k: int, group: int, dtype: int, terms: int = 0) -> float:
    terms = terms or (1 if dtype == BF16 else 3)
    return 33 * 4 * terms + (k / group + 80) / 2


def _close(got, expect, bound, dtype, what=""):
    limit = bound + HALF_STEP[dtype] * (np.abs(expect) + bound) + 1e-37
    wrong = ~(np.abs(got - expect) <= limit)
    assert not wrong.any(), (what, int(wrong.sum()), float((np.abs(got - expect) / limit).max()), np.argwhere(wrong)[:4])


def _strided(x, stride, dtype, fill=np.nan):
    """Rows `stride` apart; what lies between them is not looked at."""
    wide = np.full((x.shape[0], stride), fill, np.float32)
    wide[:, :x.shape[1]] = x
    return _bits(wide, dtype)


def _weights(seed, n, k):
    w = oracle.normal(seed, (n, k)) * np.exp2(oracle.uniform(seed + 1, (n, 1), -3.0, 3.0))
    return w.astype(np.float32)


def _matrix(dev, w, group, guard=64):
    """A packed matrix (or several) on the device, from the oracle's bytes, and the values it stands for."""
    many = w if w.ndim == 3 else w[None]
    held = [od.w4_quantise(m, group) for m in many]
    data = np.concatenate([od.w4_pack(*h, group) for h in held] + [np.full(guard, 0xEE, np.uint8)])
    values = np.stack([od.w4_values(*h, group) for h in held])
    ptr = dev.up(data)
    return p.w4_matrix(ptr, w.shape[-2], w.shape[-1], group, len(many)), (values if w.ndim == 3 else values[0])


# ------------------------------------------------------------------ packing
@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("group", (32, 64, 128))
@pytest.mark.parametrize("n,k,stride,count,lead", [
    (1, 1, 1, 1, 0), (16, 128, 128, 1, 0), (15, 127, 131, 2, 4), (17, 129, 129, 3, 0), (64, 640, 650, 1, 8),
    (5, 1000, 1000, 1, 4), (200, 33, 33, 2, 0), (3, 7, 9, 5, 4), (129, 2048, 2048, 1, 0)])
def test_packed_bytes_and_read_back(gpu_runtime, dtype, group, n, k, stride, count, lead):
    w = _rounded(_weights(n * k, count * n, k) * np.exp2(oracle.uniform(2, (count * n, 1), -30.0, 30.0)), dtype)
    held = [od.w4_quantise(m, group) for m in w.reshape(count, n, k)]
    expect = np.concatenate([od.w4_pack(*h, group) for h in held])
    values = np.concatenate([od.w4_values(*h, group) for h in held])
    with Device(gpu_runtime) as dev:
        packed = np.full(count * p.w4_bytes(n, k, group) + 32, 0xA5, np.uint8)
        ptr = dev.up(packed)
        matrix = p.w4_matrix(ptr, n, k, group, count)
        gpu_runtime.w4_pack_device(matrix, dev.up(_strided(w, stride, dtype), lead), stride, dtype)
        packed = dev.down(packed, ptr)
        out = _strided(np.full((count * n, k), -3.0), stride, dtype, -3.0)
        to = dev.up(out, lead)
        gpu_runtime.w4_unpack_device(matrix, to, stride, dtype)
        out = _values(dev.down(out, to), dtype)
    assert np.all(packed[-32:] == 0xA5) and np.array_equal(packed[:-32], expect)
    assert np.array_equal(out[:, :k].astype(np.float64), values) and np.all(out[:, k:] == -3.0)


def test_packing_borders_and_special_values(gpu_runtime):
    """Ties, zeros, the smallest and largest numbers, infinities and NaN, a group each."""
    for group in (32, 64, 128):
        x = np.zeros((9, group), np.float32)
        x[0, :9] = [6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.0]
        x[1] = np.float32(1e-45)
        x[2] = np.float32(2.0 ** -149) * np.arange(group) * 300000
        x[3] = np.linspace(-3.4e38, 3.4e38, group)
        x[4, 3] = np.inf
        x[5, 7] = np.nan
        x[6] = np.float32(2.0 ** -126) * np.linspace(-1, 1, group)
        x[7] = -0.0
        x[8] = np.exp2(np.random.default_rng(4).uniform(-30, 30, group))
        x = np.concatenate((x, -x), 1)  # two groups a row
        codes, steps = od.w4_quantise(x, group)
        with Device(gpu_runtime) as dev:
            packed = np.zeros(p.w4_bytes(9, 2 * group, group), np.uint8)
            ptr = dev.up(packed)
            matrix = p.w4_matrix(ptr, 9, 2 * group, group)
            gpu_runtime.w4_pack_device(matrix, dev.up(x), 2 * group, F32)
            packed = dev.down(packed, ptr)
            back = dev.up(np.zeros_like(x))
            gpu_runtime.w4_unpack_device(matrix, back, 2 * group, F32)
            back = dev.down(x, back)
        assert np.array_equal(packed, od.w4_pack(codes, steps, group))
        with np.errstate(over="ignore"):  # 6 s of the largest group lies past fp32's range
            assert np.array_equal(back, od.w4_values(codes, steps, group).astype(np.float32), equal_nan=True)


# ------------------------------------------------------------------ products
def _product(rt, x, w, group, dtype, x_stride=None, out_stride=None, lead=0):
    rows, k = x.shape
    n = w.shape[0]
    x_stride, out_stride = x_stride or k, out_stride or n
    with Device(rt) as dev:
        matrix, values = _matrix(dev, w, group)
        out = _strided(np.full((rows + 1, n), -7.0), out_stride, dtype, -7.0)
        to = dev.up(out, lead)
        rt.gemm_w4_device(matrix, dev.up(_strided(x, x_stride, dtype), lead), to, rows, x_stride, out_stride, dtype)
        out = _values(dev.down(out, to), dtype)
    assert np.all(out[rows] == -7.0) and np.all(out[:, n:] == -7.0)
    return out[:rows, :n].astype(np.float64), values


PRODUCTS = [
    # rows, n, k, x stride, out stride, bytes in front
    (1, 1, 1, 1, 1, 0), (1, 16, 128, 128, 16, 0), (2, 17, 129, 131, 19, 4), (3, 33, 7, 7, 33, 0), (15, 40, 255, 257, 41, 4),
    (16, 100, 640, 640, 100, 0), (17, 31, 384, 384, 31, 0), (1, 2048, 2048, 2048, 2048, 0), (1, 300, 4224, 4224, 300, 0),
    (32, 65, 520, 520, 70, 8), (33, 300, 1000, 1001, 300, 4), (48, 64, 256, 256, 64, 0), (64, 129, 1999, 1999, 131, 0),
    (5, 16, 16384, 16384, 16, 0), (31, 48, 8193, 8200, 48, 0), (65, 70, 300, 300, 70, 0), (129, 260, 513, 513, 260, 0),
    (200, 500, 640, 648, 504, 0), (300, 33, 96, 96, 33, 0), (1, 5000, 96, 96, 5000, 0)]


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("group", (32, 64, 128))
@pytest.mark.parametrize("rows,n,k,x_stride,out_stride,lead", PRODUCTS)
def test_product(gpu_runtime, dtype, group, rows, n, k, x_stride, out_stride, lead):
    x = _rounded(oracle.normal(rows + k, (rows, k)) * np.exp2(oracle.uniform(7, (rows, 1), -6.0, 6.0)), dtype)
    got, values = _product(gpu_runtime, x, _weights(n + k, n, k), group, dtype, x_stride, out_stride, lead)
    expect, size = od.product(x, values)
    _close(got, expect, _chain(k, group, dtype) * 2.0 ** -23 * size, dtype)


# Sizes at which the kernels divide the work in other ways: more columns or fewer waves a workgroup, slices of K, larger
# tiles.
DIVISIONS = [
    # rows, n, k, x stride, out stride, bytes in front
    (1, 4500, 130, 130, 4500, 0), (3, 9000, 200, 204, 9001, 4), (2, 24600, 100, 100, 24600, 0), (40, 6000, 96, 96, 6000, 0),
    (16, 700, 9000, 9000, 700, 0), (7, 2048, 8192, 8192, 2048, 0), (1, 40, 5, 5, 40, 0), (17, 4500, 6, 6, 4500, 0),
    (20, 9000, 7, 9, 9000, 4), (50, 25000, 40, 40, 25000, 0), (300, 10000, 300, 300, 10000, 0), (1024, 4000, 256, 256, 4000, 0),
    (1000, 10240, 130, 131, 10241, 4), (2049, 70, 520, 520, 70, 0), (700, 3000, 1030, 1032, 3000, 0), (1024, 520, 5, 5, 520, 0),
    (1, 24600, 128, 128, 24600, 0), (3, 9000, 256, 256, 9000, 0), (1024, 8000, 130, 130, 8000, 0), (1024, 5000, 256, 256, 5000, 0),
    (9, 4500, 131, 131, 4500, 0), (40, 9000, 128, 129, 9000, 0), (2, 24600, 100, 101, 24600, 0), (5, 600, 9001, 9001, 600, 0),
    (30, 9001, 256, 259, 9001, 0), (50, 14000, 256, 256, 14000, 0), (49, 14000, 70, 70, 14001, 0), (50, 13999, 200, 201, 13999, 0),
    (33, 3001, 199, 199, 3001, 0), (1, 10000, 131, 131, 10000, 0),
    (49, 33000, 128, 128, 33000, 0), (64, 32999, 260, 260, 32999, 0), (50, 33000, 33, 33, 33000, 0), (200, 16000, 136, 136, 16000, 0)]


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("group", (32, 64, 128))
@pytest.mark.parametrize("rows,n,k,x_stride,out_stride,lead", DIVISIONS)
def test_product_in_other_divisions(gpu_runtime, dtype, group, rows, n, k, x_stride, out_stride, lead):
    test_product(gpu_runtime, dtype, group, rows, n, k, x_stride, out_stride, lead)


@pytest.mark.parametrize("rows,k,x_stride", [(1, 8, 8), (1, 128, 128), (4, 300, 300), (20, 256, 258), (33, 1000, 1000),
                                             (20, 9, 10), (300, 640, 640)])
def test_product_of_bf16_rows_off_words(gpu_runtime, rows, k, x_stride):
    """x and out two bytes behind a word's border, rows a whole number of words apart."""
    test_product(gpu_runtime, BF16, 64, rows, 130, k, x_stride, 132, 2)


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("rows", (3, 20, 70, 200))
def test_product_of_single_ones(gpu_runtime, dtype, rows):
    """A row with a single 1 picks a weight: every column of x meets its own weight, exactly."""
    n, k = 47, 395
    w = _weights(1, n, k)
    columns = (np.arange(rows) * 53) % k
    x = np.zeros((rows, k), np.float32)
    x[np.arange(rows), columns] = 1.0
    got, values = _product(gpu_runtime, x, w, 64, dtype)
    assert np.array_equal(got, values[:, columns].T)


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("rows", (4, 70, 300))
def test_infinities_stay_in_their_rows_and_columns(gpu_runtime, dtype, rows):
    n, k = 40, 300
    x, w = _rounded(oracle.normal(1, (rows, k)), dtype), _weights(2, n, k)
    x[1, 5], x[2, 299], x[3, 7] = np.inf, np.nan, -np.inf
    w[4, 290], w[17, 0] = np.nan, np.inf
    got, values = _product(gpu_runtime, x, w, 32, dtype)
    with np.errstate(invalid="ignore"):
        expect, size = od.product(x, values)
    assert np.array_equal(np.isnan(got), np.isnan(expect))
    assert np.array_equal(got[np.isinf(expect)], expect[np.isinf(expect)]) and np.isinf(expect[1]).any()
    fine = np.isfinite(expect)
    _close(got[fine], expect[fine], _chain(k, 32, dtype) * 2.0 ** -23 * size[fine], dtype)


def test_products_of_equal_rows_have_equal_bits(gpu_runtime):
    """A row's result does not depend on its place in a call of the same size, and equal calls give equal bits."""
    for rows in (2, 16, 64, 200):
        x = _rounded(np.repeat(oracle.normal(1, (1, 700)), rows, 0), F32)
        first, _ = _product(gpu_runtime, x, _weights(3, 90, 700), 32, F32)
        again, _ = _product(gpu_runtime, x, _weights(3, 90, 700), 32, F32)
        assert np.array_equal(first, again) and np.all(first == first[0])


def test_a_product_reads_its_matrix_past_4_gib(gpu_runtime):
    """The last columns of a matrix whose codes lie past 2^32 bytes."""
    n, k, group = 131072 + 5, 1 << 16, 128
    size = p.w4_bytes(n, k, group)
    assert size > 1 << 32
    x = _rounded(oracle.normal(1, (2, k)), BF16)
    w = _weights(9, 5, k)
    codes, steps = od.w4_quantise(w, group)
    last = od.w4_pack(codes, steps, group)  # one row of tiles
    tiles_k = k // 128
    with Device(gpu_runtime) as dev:
        ptr = gpu_runtime.alloc(size)
        dev.held.append(ptr)
        gpu_runtime.upload(ptr + (n // 16) * tiles_k * 1024, last[:tiles_k * 1024])
        gpu_runtime.upload(ptr + size - tiles_k * 32, last[tiles_k * 1024:])
        out = np.zeros((2, n), np.uint16)
        to = dev.up(out)
        gpu_runtime.gemm_w4_device(p.w4_matrix(ptr, n, k, group), dev.up(_bits(x, BF16)), to, 2, k, n, BF16)
        out = _values(dev.down(out, to), BF16)[:, -5:]
    expect, sizes = od.product(x, od.w4_values(codes, steps, group))
    _close(out, expect, _chain(k, group, BF16) * 2.0 ** -23 * sizes, BF16)


# ------------------------------------------------------------------ the mixture
def _mixture(rt, case, dtype, x=None, router=None):
    tokens, hidden, inner, experts, top_k = (case[name] for name in ("tokens", "hidden", "inner", "experts", "top_k"))
    group, down_group = case.get("group", 32), case.get("down_group", case.get("group", 32))
    x_stride, out_stride = hidden + case.get("extra", 0), hidden + case.get("extra", 0) * 2
    if x is None:
        x = _rounded(oracle.normal(tokens + hidden, (tokens, hidden)), dtype)
    if router is None:
        router = (oracle.normal(5, (experts, hidden)) * (2.0 / np.sqrt(hidden))).astype(np.float32)
    gelu, renormalise = case.get("gelu", False), case.get("renormalise", False)
    lead = case.get("lead", 0)
    scale = np.float32(1.0 / np.sqrt(hidden))
    with Device(rt) as dev:
        gate, gv = _matrix(dev, oracle.normal(11, (experts, inner, hidden)) * scale * 2, group)
        up, uv = _matrix(dev, oracle.normal(12, (experts, inner, hidden)) * scale, group)
        down, dv = _matrix(dev, oracle.normal(13, (experts, hidden, inner)) * scale, down_group)
        out = _strided(np.full((tokens + 1, hidden), -7.0), out_stride, dtype, -7.0)
        to = dev.up(out, lead)
        chosen, weights = np.full(tokens * top_k + 2, -9, np.int32), np.full(tokens * top_k + 2, -9.0, np.float32)
        dc, dw = dev.up(chosen), dev.up(weights)
        rt.moe_w4_device(gate, up, down, dev.up(router), dev.up(_strided(x, x_stride, dtype), lead), to, tokens, top_k,
                         x_stride, out_stride, dtype, activation=p.MOE_GELU_TANH if gelu else p.MOE_SILU,
                         renormalise=renormalise, dexperts=dc, dweights=dw)
        out = _values(dev.down(out, to), dtype)
        chosen, weights = dev.down(chosen, dc), dev.down(weights, dw)
    assert np.all(out[tokens] == -7.0) and np.all(out[:, hidden:] == -7.0)
    assert np.all(chosen[-2:] == -9) and np.all(weights[-2:] == -9.0)
    chosen, weights = chosen[:-2].reshape(tokens, top_k), weights[:-2].reshape(tokens, top_k)
    expect_chosen, expect_weights = od.route(x, router, top_k, renormalise)
    assert np.array_equal(chosen, expect_chosen)
    assert np.allclose(weights, expect_weights, rtol=2.0 ** -22, atol=1e-37, equal_nan=True)
    chain = max(_chain(hidden, group, dtype), _chain(inner, down_group, dtype, 2 if dtype == BF16 else 3))
    expect, bound = od.mixture(x, chosen, weights.astype(np.float64), gv, uv, dv, gelu, chain,
                               2.0 ** -16 if dtype == BF16 else 2.0 ** -24)
    return out[:tokens, :hidden].astype(np.float64), expect, bound


MIXTURES = [
    dict(tokens=1, hidden=128, inner=64, experts=4, top_k=2),
    dict(tokens=1, hidden=1, inner=1, experts=1, top_k=1),
    dict(tokens=1, hidden=300, inner=70, experts=9, top_k=9, group=64, gelu=True),
    dict(tokens=2, hidden=256, inner=128, experts=70, top_k=8, group=128, renormalise=True),
    dict(tokens=5, hidden=650, inner=129, experts=3, top_k=3, group=64, down_group=32, gelu=True, extra=3, lead=4),
    dict(tokens=16, hidden=130, inner=33, experts=2, top_k=1, renormalise=True),
    dict(tokens=17, hidden=96, inner=250, experts=8, top_k=2, group=128, gelu=True),
    dict(tokens=40, hidden=64, inner=16, experts=2, top_k=2),
    dict(tokens=64, hidden=200, inner=100, experts=16, top_k=4, group=64, renormalise=True, extra=1),
    dict(tokens=65, hidden=128, inner=48, experts=1, top_k=1),
    dict(tokens=150, hidden=64, inner=40, experts=3, top_k=2, group=64, gelu=True),
    dict(tokens=3, hidden=64, inner=32, experts=1024, top_k=64),
    dict(tokens=1, hidden=1024, inner=1100, experts=6, top_k=3, group=32, gelu=True, renormalise=True),
]


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("index", range(len(MIXTURES)))
def test_mixture(gpu_runtime, index, dtype):
    _close(*_mixture(gpu_runtime, MIXTURES[index], dtype), dtype)


# As above: parts of K with one block of pairs and with several, wide output columns, lists of pairs, blocks taken at once,
# output columns joined in a launch of their own, rows shorter than eight.
MIXTURE_DIVISIONS = [
    dict(tokens=8, hidden=64, inner=600, experts=24, top_k=2, group=64),
    dict(tokens=16, hidden=100, inner=2100, experts=5, top_k=3, gelu=True),
    dict(tokens=20, hidden=96, inner=1030, experts=8, top_k=2, group=128, renormalise=True),
    dict(tokens=64, hidden=48, inner=520, experts=4, top_k=4, group=64),
    dict(tokens=64, hidden=256, inner=130, experts=64, top_k=8, renormalise=True, extra=3, lead=4),
    dict(tokens=33, hidden=70, inner=48, experts=100, top_k=2, group=128),
    dict(tokens=64, hidden=40, inner=20, experts=300, top_k=9, group=64, gelu=True),
    dict(tokens=3, hidden=7, inner=5, experts=6, top_k=2),
    dict(tokens=66, hidden=6, inner=200, experts=70, top_k=3, group=64, down_group=128),
    dict(tokens=2, hidden=33000, inner=24, experts=2, top_k=1, gelu=True),
    dict(tokens=100, hidden=130, inner=70, experts=80, top_k=4, group=64, extra=1),
    dict(tokens=1000, hidden=64, inner=140, experts=4, top_k=2, group=128, gelu=True),
    dict(tokens=520, hidden=33, inner=24, experts=200, top_k=1, renormalise=True),
    dict(tokens=3, hidden=131, inner=40, experts=3, top_k=1, group=128),
    dict(tokens=70, hidden=129, inner=40, experts=3, top_k=1, group=128, gelu=True),
]


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("index", range(len(MIXTURE_DIVISIONS)))
def test_mixture_in_other_divisions(gpu_runtime, index, dtype):
    _close(*_mixture(gpu_runtime, MIXTURE_DIVISIONS[index], dtype), dtype)


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("group", (32, 64, 128))
@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", [
    (1, 5, 3, 70, 2), (70, 6, 130, 3, 2), (1, 128, 20, 300, 3), (4, 130, 1200, 6, 2), (1, 256, 128, 3, 1), (80, 384, 40, 2, 1)])
def test_mixture_of_every_group(gpu_runtime, dtype, group, tokens, hidden, inner, experts, top_k):
    case = dict(tokens=tokens, hidden=hidden, inner=inner, experts=experts, top_k=top_k, group=group)
    _close(*_mixture(gpu_runtime, case, dtype), dtype)


def test_mixtures_of_equal_calls_have_equal_bits(gpu_runtime):
    for tokens in (1, 12, 64, 200):
        case = dict(tokens=tokens, hidden=200, inner=600, experts=12, top_k=5)
        first, again = (_mixture(gpu_runtime, case, F32)[0] for _ in range(2))
        assert np.array_equal(first, again)


@pytest.mark.parametrize("tokens", (1, 3, 30))
def test_mixture_ties_go_to_the_lower_expert(gpu_runtime, tokens):
    """Equal logits (experts with equal router rows), and a token of zeros, whose logits are all equal."""
    case = dict(tokens=tokens, hidden=96, inner=32, experts=80, top_k=6, renormalise=True)
    x = _rounded(oracle.normal(3, (tokens, 96)), F32)
    x[0] = 0.0
    router = np.repeat(oracle.normal(4, (20, 96)), 4, 0)[np.random.default_rng(1).permutation(80)]
    _close(*_mixture(gpu_runtime, case, F32, x, router), F32)


def test_mixture_all_tokens_to_one_expert(gpu_runtime):
    for tokens in (16, 33, 64, 130):
        case = dict(tokens=tokens, hidden=64, inner=32, experts=5, top_k=1)
        x = _rounded(np.abs(oracle.normal(3, (tokens, 64))), BF16)
        router = np.zeros((5, 64), np.float32)
        router[3] = 1.0
        _close(*_mixture(gpu_runtime, case, BF16, x, router), BF16)


def test_mixture_nan_and_infinities_stay_in_their_tokens(gpu_runtime):
    case = dict(tokens=20, hidden=128, inner=64, experts=6, top_k=2)
    for dtype in (F32, BF16):
        x = _rounded(oracle.normal(3, (20, 128)), dtype)
        x[4, 7], x[11, 100], x[12] = np.nan, np.inf, np.nan
        rt = gpu_runtime
        router = (oracle.normal(5, (6, 128)) * 0.2).astype(np.float32)
        with np.errstate(invalid="ignore"):
            got, expect, bound = _mixture_loose(rt, case, dtype, x, router)
        fine = np.ones(20, bool)
        fine[[4, 11, 12]] = False
        assert np.isnan(got[[4, 11, 12]]).all()
        _close(got[fine], expect[fine], bound[fine], dtype)


def _mixture_loose(rt, case, dtype, x, router):
    """As _mixture; the oracle's rows of NaN are compared by the caller."""
    with np.errstate(all="ignore"):
        return _mixture(rt, case, dtype, x, router)


# ------------------------------------------------------------------ rotary positions
ROPES = [
    # rows, head dim, rotary, pairs, q heads, k heads
    (1, 64, 64, False, 4, 1), (3, 128, 64, True, 3, 2), (5, 80, 20, False, 2, 0), (2, 80, 80, True, 0, 5),
    (7, 256, 256, False, 8, 1), (4, 2, 2, True, 1, 1), (4, 10, 6, False, 3, 1), (9, 96, 2, False, 2, 2),
    (2, 1024, 1024, True, 1, 1), (300, 128, 128, False, 5, 1), (33, 72, 40, True, 4, 4), (2, 64, 16, False, 70, 1)]


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("in_place", (False, True))
@pytest.mark.parametrize("index", range(len(ROPES)))
def test_rope(gpu_runtime, index, in_place, dtype):
    rows, dim, rotary, pairs, q_heads, k_heads = ROPES[index]
    rng = np.random.default_rng(index)
    positions = rng.integers(0, 200000, rows).astype(np.int32)
    positions[0] = (0, -17, 2 ** 31 - 1, -2 ** 31)[index % 4]
    turns, magnitude = p.rope_turns(rotary, 10000.0, p.ROPE_SCALE_PARTS if index % 2 else 0, 8.0, 4096.0)
    with Device(gpu_runtime) as dev:
        made = []
        for heads, extra in ((q_heads, 5), (k_heads, 0)):
            if heads == 0:
                made.append((None, None, None))
                continue
            x = _rounded(oracle.normal(heads + rows, (rows, heads * dim)), dtype)
            stride, out_stride = heads * dim + extra, heads * dim + (extra if in_place else 3)
            lead = 4 if extra else 0
            source = dev.up(_strided(x, stride, dtype, -7.0), lead)
            out = _strided(np.full_like(x, -7.0), out_stride, dtype, -7.0)
            to = source if in_place else dev.up(out, lead)
            made.append(((source, to, heads, stride, out_stride), x.reshape(rows, heads, dim), out))
        gpu_runtime.rope_device(dev.up(positions), dev.up(turns), rows, dim, rotary, p.ROPE_PAIRS if pairs else p.ROPE_HALF,
                                dtype, magnitude, made[0][0], made[1][0])
        for call, x, out in made:
            if call is None:
                continue
            got = _values(dev.down(out, call[1]), dtype)
            width = call[2] * dim
            assert np.all(got[:, width:] == -7.0)
            got = got[:, :width].reshape(x.shape).astype(np.float64)
            expect, bound = od.rope(x, positions, turns, rotary, pairs, magnitude)
            assert np.array_equal(got[..., rotary:], x[..., rotary:])
            _close(got, expect, bound, dtype)


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("rows,dim,rotary,pairs,q_heads,k_heads", [
    (4099, 64, 32, False, 5, 1), (4096, 64, 64, True, 3, 2), (5001, 10, 6, False, 3, 1), (4097, 6, 4, True, 1, 1),
    (4102, 1024, 16, False, 1, 0), (4100, 80, 40, False, 3, 1), (4099, 80, 20, False, 2, 2), (4097, 80, 20, True, 2, 2),
    (4098, 12, 2, True, 3, 1), (4097, 7, 4, False, 3, 1), (3, 80, 40, False, 3, 1), (5, 22, 20, False, 2, 1),
    (3, 80, 20, True, 3, 1), (3, 20, 18, True, 2, 1), (2, 9, 4, True, 5, 1), (300, 9, 6, False, 5, 1),
    (4098, 9, 4, True, 3, 1)])
def test_rope_in_other_divisions(gpu_runtime, rows, dim, rotary, pairs, q_heads, k_heads, dtype, monkeypatch):
    monkeypatch.setitem(globals(), "ROPES", [(rows, dim, rotary, pairs, q_heads, k_heads)])
    for in_place in (False, True):
        test_rope(gpu_runtime, 0, in_place, dtype)


def test_rope_back_to_where_it_was(gpu_runtime):
    """The opposite position turns back: a rotation of far positions loses only roundings."""
    x = oracle.normal(1, (2, 128))
    turns, _ = p.rope_turns(128)
    with Device(gpu_runtime) as dev:
        to = dev.up(x)
        for position in (1234567, -1234567):
            gpu_runtime.rope_device(dev.up(np.full(2, position, np.int32)), dev.up(turns), 2, 128, 128, p.ROPE_HALF, F32,
                                    q=(to, to, 1, 128, 128))
        got = dev.down(x, to)
    # twice the bound of one rotation (angle 2^-26 turns, nine roundings) times |a| + |b| <= 2 max |x|
    assert np.abs(got - x).max() <= 2 * 2 * np.abs(x).max() * (2 * np.pi * 2.0 ** -26 + 12 * 2.0 ** -24)


# ------------------------------------------------------------------ residual sums with norms
NORMS = [dict(rows=1, width=1), dict(rows=3, width=7, extra=2, lead=4), dict(rows=5, width=64), dict(rows=9, width=512),
         dict(rows=2, width=513, extra=1), dict(rows=1, width=2048), dict(rows=3, width=2049), dict(rows=2, width=4096),
         dict(rows=4, width=4100, extra=5, lead=4), dict(rows=3, width=8192), dict(rows=2, width=10000),
         dict(rows=2, width=16385), dict(rows=1, width=32768), dict(rows=700, width=130, per=9)]
PARTS = [dict(), dict(y=1), dict(y=1, post=1, pre=1), dict(y=1, gate=1, pre=1, scale=1, shift=1), dict(scale=1, pre=1),
         dict(y=1, post=1, gate=1, tanh=1, pre=1, scale=1, shift=1, offset=1.0, residual=0.25, in_place=1),
         dict(y=1, post=1, no_out=1), dict(y=1, gate=1, tanh=1, no_h=1, shift=1, in_place=1)]


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("parts", range(len(PARTS)))
@pytest.mark.parametrize("index", range(len(NORMS)))
def test_residual_norm(gpu_runtime, index, parts, dtype):
    case, has = NORMS[index], PARTS[parts]
    rows, width, extra, lead = case["rows"], case["width"], case.get("extra", 0), case.get("lead", 0)
    per = case.get("per", 2)
    stride, vector_stride = width + extra, 2 * width + extra
    shared = -(-rows // per)
    h, y = (_rounded(oracle.normal(index + i, (rows, width)) * s, dtype) for i, s in ((1, 3.0), (2, 0.7)))
    vectors = {name: _rounded(oracle.normal(index + i, (shared, width)), dtype)
               for i, name in enumerate(("gate", "scale", "shift")) if has.get(name)}
    weights = {name: (oracle.normal(i, (width,)) * 0.1 + 1.0).astype(np.float32)
               for i, name in enumerate(("post", "pre")) if has.get(name)}
    keep = dict(gate_tanh=bool(has.get("tanh")), rows_per_vector=per, residual_scale=has.get("residual", 1.0),
                weight_offset=has.get("offset", 0.0), eps=1e-5)
    expect_h, expect, bound_h, bound = od.residual_norm(h, y if has.get("y") else None, **vectors, **weights, **keep)
    with Device(gpu_runtime) as dev:
        blank = _strided(np.full_like(h, -7.0), stride, dtype, -7.0)
        dh, dy = dev.up(_strided(h, stride, dtype, -7.0), lead), dev.up(_strided(y, stride, dtype, -7.0), lead)
        to_h = None if has.get("no_h") else dh if has.get("in_place") else dev.up(blank, lead)
        to = None if has.get("no_out") else dy if has.get("in_place") else dev.up(blank)
        on = {"d" + name: dev.up(_strided(v, vector_stride, dtype), lead) for name, v in vectors.items()}
        on.update({"d" + name: dev.up(v, 4 if lead else 0) for name, v in weights.items()})
        gpu_runtime.residual_norm_device(dh, to_h, to, rows, width, dtype, dy=dy if has.get("y") else None, **on, **keep,
                                         h_stride=stride, y_stride=stride, h_out_stride=stride, out_stride=stride,
                                         vector_stride=vector_stride)
        for ptr, value, limit in ((to_h, expect_h, bound_h), (to, expect, bound)):
            if ptr is not None:
                got = _values(dev.down(blank, ptr), dtype)
                assert np.all(got[:, width:] == -7.0)
                _close(got[:, :width].astype(np.float64), value, limit, dtype)


# Enough rows that a workgroup takes several, with vectors that change between them.
MANY_NORMS = [dict(rows=9001, width=40, per=9), dict(rows=2500, width=600, per=7), dict(rows=4500, width=600, per=7),
              dict(rows=4099, width=1001, per=2),
              dict(rows=2500, width=1504, per=3), dict(rows=2100, width=1501, per=4), dict(rows=1300, width=2056, per=500),
              dict(rows=1201, width=4099, per=1, extra=1, lead=4), dict(rows=600, width=8200, per=77),
              dict(rows=600, width=8201, per=77),
              dict(rows=600, width=16400, per=600)]


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("parts", (0, 2, 3, 5, 6))
@pytest.mark.parametrize("index", range(len(MANY_NORMS)))
def test_residual_norm_of_many_rows(gpu_runtime, index, parts, dtype, monkeypatch):
    monkeypatch.setitem(globals(), "NORMS", MANY_NORMS)
    test_residual_norm(gpu_runtime, index, parts, dtype)


def test_residual_norm_of_extreme_rows(gpu_runtime):
    """Squares past fp32's range, below it, rows of zeros, and NaN that stays in its row."""
    x = oracle.normal(1, (6, 600))
    x[0] *= np.float32(1e30)
    x[1] *= np.float32(1e-30)
    x[2] = 0.0
    x[3, 5] = np.nan
    x[4, 9] = np.inf
    with Device(gpu_runtime) as dev:
        to = dev.up(np.zeros_like(x))
        gpu_runtime.residual_norm_device(dev.up(x), None, to, 6, 600, F32, eps=0.0)
        got = dev.down(x, to)
    wide = x.astype(np.float64)
    for row in (0, 1, 5):
        expect = wide[row] / np.sqrt((wide[row] ** 2).mean())
        assert np.all(np.abs(got[row] - expect) <= 4 * 2.0 ** -24 * np.abs(expect) + 1e-37)
    assert np.isnan(got[2:4]).all()  # 0 / 0 without an eps
    assert np.isnan(got[4, 9]) and np.all(got[4, :9] == 0.0)


# ------------------------------------------------------------------ together
def test_a_decoder_step(gpu_runtime):
    """A layer's step for two conversations: norm, projections, positions, the cache, attention, projection, residual
    norm, mixture, residual: queued without a wait, each stage held to its definition on what the one before left."""
    rt, dtype = gpu_runtime, BF16
    hidden, heads, kv_heads, dim, inner, experts, top_k, rows = 256, 4, 2, 64, 96, 8, 2, 2
    lengths = np.array([70, 5], np.int32)  # the new token among them
    width, kv_width = heads * dim, kv_heads * dim
    total = width + 2 * kv_width
    block = p.kv4_page_bytes(dim, kv_heads)
    rng = np.random.default_rng(8)
    h0 = _rounded(oracle.normal(1, (rows, hidden)), dtype)
    norms = [(oracle.normal(i, (hidden,)) * 0.1 + 1.0).astype(np.float32) for i in range(3)]
    small = np.float32(1.0 / np.sqrt(hidden))
    turns, magnitude = p.rope_turns(dim)
    positions = lengths - 1
    pages, table = 4, np.array([[2, 0], [3, -1]], np.int32)
    caches = oq.Cache(pages, kv_heads, dim, np.zeros((pages, kv_heads, 64 * dim + 4 * dim), np.uint8))
    for seq in range(rows):
        for t in range(lengths[seq] - 1):
            caches.store(table[seq, t // 64], t % 64, rng.standard_normal((kv_heads, dim)).astype(np.float32),
                         rng.standard_normal((kv_heads, dim)).astype(np.float32))
    router = (oracle.normal(5, (experts, hidden)) * 0.3).astype(np.float32)
    with Device(rt) as dev:
        blank = lambda w: dev.up(np.zeros((rows, w), np.uint16))  # noqa: E731
        qkv, qkv_values = _matrix(dev, oracle.normal(21, (total, hidden)) * small, 64)
        proj, proj_values = _matrix(dev, oracle.normal(22, (hidden, width)) * small, 128)
        gate, gv = _matrix(dev, oracle.normal(23, (experts, inner, hidden)) * small, 32)
        up, uv = _matrix(dev, oracle.normal(24, (experts, inner, hidden)) * small, 32)
        down, dv = _matrix(dev, oracle.normal(25, (experts, hidden, inner)) * small, 32)
        assert block == kv_heads * caches.block
        pool, dtable, dlengths = dev.up(caches.pool), dev.up(table), dev.up(lengths)
        starts = dev.up(np.array([0, 1, 2], np.int32))
        cache = p.kv4_cache(pool, dtable, dlengths, dim, kv_heads, pages, rows, 2)
        h = dev.up(_bits(h0, dtype))
        x, packed, turned, seen, o, h1, x1, moe, h2, x2 = (blank(w) for w in (
            hidden, total, total, width, hidden, hidden, hidden, hidden, hidden, hidden))
        chosen, weights = dev.up(np.zeros((rows, top_k), np.int32)), dev.up(np.zeros((rows, top_k), np.float32))
        dnorms = [dev.up(n) for n in norms]
        dpositions, dturns = dev.up(positions.astype(np.int32)), dev.up(turns)
        drouter = dev.up(router)
        rt.residual_norm_device(h, None, x, rows, hidden, dtype, dpre=dnorms[0])
        rt.gemm_w4_device(qkv, x, packed, rows, hidden, total, dtype)
        rt.rope_device(dpositions, dturns, rows, dim, dim, p.ROPE_HALF, dtype, magnitude,
                       q=(packed, turned, heads, total, total),
                       k=(packed + 2 * width, turned + 2 * width, kv_heads, total, total))
        rt.kv4_write_device(cache, turned + 2 * width, packed + 2 * (width + kv_width), starts, rows, total, dtype)
        rt.attention_kv4_device(cache, turned, seen, starts, rows, heads, total, width, 1, 70, 0, dim ** -0.5, dtype)
        rt.gemm_w4_device(proj, seen, o, rows, width, hidden, dtype)
        rt.residual_norm_device(h, h1, x1, rows, hidden, dtype, dy=o, dpost=dnorms[1], dpre=dnorms[2])
        rt.moe_w4_device(gate, up, down, drouter, x1, moe, rows, top_k, hidden, hidden, dtype, renormalise=True,
                         dexperts=chosen, dweights=weights)
        rt.residual_norm_device(h1, h2, x2, rows, hidden, dtype, dy=moe, dpre=dnorms[0])
        get = lambda ptr, w: _values(dev.down(np.zeros((rows, w), np.uint16), ptr), dtype)  # noqa: E731
        x, packed, turned, seen, o, h1, x1, moe, h2, x2 = (get(*pair) for pair in (
            (x, hidden), (packed, total), (turned, total), (seen, width), (o, hidden), (h1, hidden), (x1, hidden),
            (moe, hidden), (h2, hidden), (x2, hidden)))
        chosen = dev.down(np.zeros((rows, top_k), np.int32), chosen)
        weights = dev.down(np.zeros((rows, top_k), np.float32), weights)
    _, expect, _, bound = od.residual_norm(h0, pre=norms[0])
    _close(x, expect, bound, dtype, "norm")
    expect, size = od.product(x, qkv_values)
    _close(packed, expect, _chain(hidden, 64, dtype) * 2.0 ** -23 * size, dtype, "projections")
    for first, count in ((0, heads), (width, kv_heads)):
        part = slice(first, first + count * dim)
        expect, bound = od.rope(packed[:, part].reshape(rows, count, dim), positions, turns, dim, False, magnitude)
        _close(turned[:, part].reshape(rows, count, dim), expect, bound, dtype, "positions")
    keys, values = turned[:, width:width + kv_width], packed[:, width + kv_width:]
    rng = np.random.default_rng(8)
    for seq in range(rows):
        held_k, held_v = [], []
        for t in range(lengths[seq]):
            if t < lengths[seq] - 1:
                k, v = (rng.standard_normal((kv_heads, dim)).astype(np.float32) for _ in range(2))
            else:
                k, v = keys[seq].reshape(kv_heads, dim), values[seq].reshape(kv_heads, dim)
            held_k.append(oq.kv4_values(*oq.kv4_quantise(k)))
            held_v.append(oq.kv4_values(*oq.kv4_quantise(v)))
        out, size, reach = oq.attention(turned[seq, :width].reshape(heads, dim).astype(np.float64), np.stack(held_k),
                                        np.stack(held_v), int(positions[seq]), dim ** -0.5)
        bound = (2.0 ** -8 + 2.0 ** -16 + (4 * (dim + 16) * reach[:, None] + 200) * 2.0 ** -24) * size
        _close(seen[seq].reshape(heads, dim), out, bound, dtype, "attention")
    expect, size = od.product(seen, proj_values)
    _close(o, expect, _chain(width, 128, dtype) * 2.0 ** -23 * size, dtype, "projection")
    expect_h, expect, bound_h, bound = od.residual_norm(h0, o, post=norms[1], pre=norms[2])
    _close(h1, expect_h, bound_h, dtype, "residual")
    _close(x1, expect, bound, dtype, "residual norm")
    expect_chosen, expect_weights = od.route(x1, router, top_k, True)
    assert np.array_equal(chosen, expect_chosen) and np.allclose(weights, expect_weights, rtol=2.0 ** -22)
    chain = max(_chain(hidden, 32, dtype), _chain(inner, 32, dtype, 2))
    expect, bound = od.mixture(x1, chosen, weights.astype(np.float64), gv, uv, dv, False, chain, 2.0 ** -16)
    _close(moe, expect, bound, dtype, "mixture")
    expect_h, expect, bound_h, bound = od.residual_norm(h1, moe, pre=norms[0])
    _close(h2, expect_h, bound_h, dtype, "second residual")
    _close(x2, expect, bound, dtype, "last norm")


def test_calls_that_share_the_workspace(gpu_runtime):
    """Mixtures and sliced products of different sizes, queued one behind the other and from two threads, give what
    each gives alone."""
    rt = gpu_runtime
    with Device(rt) as dev:
        jobs = []
        for tokens, hidden, inner, experts in ((1, 512, 256, 6), (40, 256, 64, 12), (3, 128, 640, 4)):
            gate, _ = _matrix(dev, oracle.normal(1, (experts, inner, hidden)), 32)
            up, _ = _matrix(dev, oracle.normal(2, (experts, inner, hidden)), 32)
            down, _ = _matrix(dev, oracle.normal(3, (experts, hidden, inner)), 64)
            x, router = dev.up(oracle.normal(4, (tokens, hidden))), dev.up(oracle.normal(5, (experts, hidden)))
            out = np.zeros((tokens, hidden), np.float32)
            to = [dev.up(out) for _ in range(9)]
            jobs.append((out, to, lambda i, a=(gate, up, down, router, x), to=to, t=tokens, h=hidden: rt.moe_w4_device(
                *a, to[i], t, 3, h, h, F32)))
        for rows, n, k in ((4, 64, 16384), (40, 128, 8192)):
            matrix, _ = _matrix(dev, _weights(6, n, k), 64)
            x = dev.up(oracle.normal(7, (rows, k)))
            out = np.zeros((rows, n), np.float32)
            to = [dev.up(out) for _ in range(9)]
            jobs.append((out, to, lambda i, a=(matrix, x), to=to, r=rows, n=n, k=k: rt.gemm_w4_device(*a, to[i], r, k, n, F32)))
        for _, _, job in jobs:
            job(0)
            rt.synchronize()
        for i in (1, 2):
            for _, _, job in jobs:
                job(i)
        threads = [threading.Thread(target=lambda first=first: [job(i) for i in range(first, first + 3) for _, _, job in jobs])
                   for first in (3, 6)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for out, to, _ in jobs:
            first = dev.down(out, to[0])
            assert np.isfinite(first).all() and first.any()
            for other in to[1:]:
                assert np.array_equal(dev.down(out, other), first)
