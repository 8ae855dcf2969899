"""The quantised decode path on the GPU against its definitions in 64 bits (oracle/quantised.py).

Quantised rows, cache pages and what is read back are compared bit for bit.  Tolerances:

product: an exact int32 sum goes through one rounding to fp32 and two products, each at most
2^-24 of the value: 3 * 2^-24, and for bf16 results half a step (2^-8) more.

attention: scores are fp32 sums of D exact terms, so off by at most (D + 16) 2^-24 of
A = scale * sum_d |q_d k_td| (16: the groups' steps, the scale and the exponent's argument),
which changes each probability, its weight and their sum by twice that; exp and the rounded
maximum add 2^-21; sums over T tokens in fp32 add at most (T / 16 + 64) 2^-24 of
W = sum_t p_t |v_t| (T / 16: the longest chain of additions in a lane).  Probabilities enter
the product with 24 bits (fp32) or at least 8 (bf16: 2^-8 of W), and the result is rounded
once (2^-24, 2^-8 of it)."""
from __future__ import annotations

import numpy as np
import pytest

import oracle
from oracle import quantised as oq
from oct_amd import prometheus as p
from tests.test_quantised_path import PLANNED, smallest_rows

pytestmark = pytest.mark.gpu

F32, BF16 = p.DTYPE_F32, p.DTYPE_BF16


class Device:
    """Device copies of numpy arrays, freed at the end."""

    def __init__(self, rt):
        self.rt, self.held = rt, []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.rt.synchronize()
        for ptr in self.held:
            self.rt.free(ptr)

    def up(self, array, lead: int = 0) -> int:
        """A copy of `array`, `lead` bytes behind an aligned address."""
        array = np.ascontiguousarray(array)
        ptr = self.rt.alloc(array.nbytes + lead + 64)
        self.held.append(ptr)
        self.rt.upload(ptr + lead, array)
        return ptr + lead

    def down(self, like, ptr: int):
        self.rt.synchronize()
        return self.rt.download(np.empty(like.shape, like.dtype), ptr)


def _bits(x, dtype):
    return oracle.to_bf16(x) if dtype == BF16 else np.ascontiguousarray(x, np.float32)


def _values(bits, dtype):
    return oracle.from_bf16(bits) if dtype == BF16 else bits


def _rounded(x, dtype):
    return _values(_bits(x, dtype), dtype)


# ------------------------------------------------------------------ rows in 8 bits
def _quantise_rows(rt, x, dtype, stride=None, lead=0):
    rows, width = x.shape
    stride = stride or width
    wide = np.full((rows, stride), np.nan, np.float32)  # what lies between rows is not looked at
    wide[:, :width] = x
    with Device(rt) as dev:
        dx = dev.up(_bits(wide, dtype), lead)
        q = np.full((rows * width + 16,), 77, np.int8)
        s = np.full((rows + 4,), -5.0, np.float32)
        dq, ds = dev.up(q, lead), dev.up(s)
        rt.quantize_rows_int8_device(dx, dq, ds, rows, width, stride, dtype)
        q, s = dev.down(q, dq), dev.down(s, ds)
    assert np.all(q[rows * width:] == 77) and np.all(s[rows:] == -5.0)
    return q[:rows * width].reshape(rows, width), s[:rows]


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("rows,width,stride,lead", [
    (1, 1, 1, 0), (3, 7, 7, 0), (5, 8, 11, 4), (4, 63, 64, 0), (9, 512, 512, 0), (2, 513, 513, 8), (3, 1024, 1027, 4),
    (1, 2048, 2048, 0), (3, 2049, 2050, 12), (2, 4097, 4097, 0), (2, 8192, 8192, 0), (3, 8193, 8200, 4),
    (2, 16384, 16384, 0), (2, 16385, 16385, 4), (1, 70001, 70001, 0), (1030, 130, 131, 0)])
def test_rows_equal_the_definition(gpu_runtime, dtype, rows, width, stride, lead):
    x = _rounded(oracle.normal(rows + width, (rows, width)) * np.exp2(oracle.uniform(9, (rows, 1), -20, 20)), dtype)
    q, s = _quantise_rows(gpu_runtime, x, dtype, stride, lead)
    eq, es = oq.quantize_rows(x)
    assert np.array_equal(s, es)
    assert np.array_equal(q, eq)


def test_rows_at_borders_and_special_values(gpu_runtime):
    """Halves of a step, zeros, the smallest and largest numbers, infinities and NaN."""
    x = np.zeros((10, 160), np.float32)
    x[0, :100] = np.arange(100) + 0.5  # with the scale 1 of the largest: ties
    x[0, 159] = 127.0
    x[1] = 0.0
    x[2, 5] = np.float32(1e-45)  # a row of one subnormal: its scale rounds to 0
    x[3, :50] = np.float32(2.0 ** -149) * np.arange(0, 25400, 508)
    x[4] = np.linspace(-3.4e38, 3.4e38, 160)
    x[5, 7] = np.inf
    x[6, 9] = np.nan
    x[7, 11], x[7, 12] = -np.inf, np.nan
    x[8] = -0.0
    x[9] = np.float32(2.0 ** -126) * np.linspace(-1, 1, 160)
    q, s = _quantise_rows(gpu_runtime, x, F32)
    eq, es = oq.quantize_rows(x)
    assert np.array_equal(s, es, equal_nan=True)
    assert np.array_equal(q, eq)


def test_rows_of_the_smallest_numbers(gpu_runtime):
    x, q, scale = smallest_rows()
    got, got_scale = _quantise_rows(gpu_runtime, x, F32)
    assert np.array_equal(got_scale, scale)
    assert np.array_equal(got, q)


def _beside(x):
    """x and its four nearest fp32 neighbours, on a last axis."""
    bits = np.ascontiguousarray(x, np.float32).view(np.int32)
    return np.stack([bits + d for d in (-2, -1, 0, 1, 2)], -1).view(np.float32)


@pytest.mark.parametrize("power", (-120, -91, -60, 0, 60, 89, 110))
def test_rows_next_to_where_rounding_changes(gpu_runtime, power):
    """Values within two ulps of every half step, of scales of any significand."""
    rng = np.random.default_rng(power + 200)
    x = np.zeros((64, 640), np.float32)
    top = (rng.uniform(1, 2, 64) * 2.0 ** power).astype(np.float32)
    scale = (top / np.float32(127.0)).astype(np.float32)
    halves = (np.arange(127) + 0.5).astype(np.float32)
    x[:, :635] = _beside(scale[:, None] * halves).reshape(64, -1) * rng.choice([-1, 1], (64, 635))
    x = np.where(np.abs(x) > top[:, None], np.float32(0.0), x)
    x[:, 639] = top
    q, s = _quantise_rows(gpu_runtime, x, F32)
    eq, es = oq.quantize_rows(x)
    assert np.array_equal(s, es) and np.array_equal(q, eq)


# ------------------------------------------------------------------ the product
def _product(rt, a, w, sa, sw, dtype, lead=0):
    (m, k), n = a.shape, w.shape[0]
    out = np.full((m * n + 8,), 0x7FC1 if dtype == BF16 else np.float32(np.nan), np.uint16 if dtype == BF16 else np.float32)
    with Device(rt) as dev:
        dc = dev.up(out)
        rt.gemm_int8_device(dev.up(a, lead), dev.up(w, lead), dev.up(sa), dev.up(sw), dc, m, n, k, dtype)
        out = dev.down(out, dc)
    tail = out[m * n:]
    assert np.all(tail == 0x7FC1) if dtype == BF16 else np.all(np.isnan(tail))
    return _values(out[:m * n].reshape(m, n), dtype)


def _check_product(got, a, w, sa, sw, dtype):
    ref = oq.int8_product(a, w, sa, sw)
    tol = (3 * 2.0 ** -24 + (2.0 ** -8 if dtype == BF16 else 0.0)) * np.abs(ref) * (1 + 2.0 ** -7)
    bad = np.abs(got.astype(np.float64) - ref) > tol
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist())


def _whole(seed, shape, low=-127, high=127):
    return np.random.default_rng(seed).integers(low, high + 1, shape, dtype=np.int8)


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 33, 15), (1, 16, 64), (1, 2048, 2048), (2, 100, 257), (15, 129, 1000), (16, 16400, 256), (17, 40, 640),
    (32, 1000, 8191), (33, 64, 128), (33, 65, 129), (64, 64, 16), (65, 130, 4096), (100, 3000, 48), (129, 257, 511),
    (257, 300, 1040), (513, 520, 2048), (700, 1100, 385), (1030, 2050, 272)])
def test_product_equals_the_exact_sums(gpu_runtime, m, n, k, dtype):
    a, w = _whole(m + k, (m, k)), _whole(n + k, (n, k), -128)
    sa, sw = oracle.uniform(1, (m,), 0.001, 0.03), oracle.uniform(2, (n,), -0.001, 0.001)
    _check_product(_product(gpu_runtime, a, w, sa, sw, dtype), a, w, sa, sw, dtype)


@pytest.mark.parametrize("m,n,k,lead", [(3, 50, 640, 1), (48, 100, 640, 8), (300, 200, 512, 3), (40, 4100, 77, 5)])
def test_product_of_operands_at_any_address(gpu_runtime, m, n, k, lead):
    a, w = _whole(5, (m, k)), _whole(6, (n, k))
    sa, sw = oracle.uniform(3, (m,), 0.001, 0.03), oracle.uniform(4, (n,), 0.0001, 0.001)
    _check_product(_product(gpu_runtime, a, w, sa, sw, F32, lead), a, w, sa, sw, F32)


@pytest.mark.parametrize("m,n", [(1, 20), (20, 20), (40, 70)])
def test_product_at_the_largest_sum(gpu_runtime, m, n):
    """-128 * -128 * 131071 is 2^31 - 2^14: the last sum that 32 bits hold."""
    k = p.GEMM_INT8_MAX_K
    a, w = np.full((m, k), -128, np.int8), np.full((n, k), -128, np.int8)
    w[n // 2:] = 127
    one = np.ones(max(m, n), np.float32)
    _check_product(_product(gpu_runtime, a, w, one[:m], one[:n], F32), a, w, one[:m], one[:n], F32)


def test_product_of_rows_that_were_not_finite_is_nan(gpu_runtime):
    for m in (5, 200):
        a, w = _whole(7, (m, 256)), _whole(8, (90, 256))
        a[2] = 0
        sa, sw = np.full(m, 0.5, np.float32), np.full(90, 0.25, np.float32)
        sa[2] = np.nan
        got = _product(gpu_runtime, a, w, sa, sw, BF16)
        assert np.isnan(got[2]).all() and np.isfinite(np.delete(got, 2, 0)).all()


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("m,n,k", [
    # few rows: 4, 8 and 16 waves a workgroup, one and two blocks of rows
    (2, 17000, 4100), (16, 5000, 5000), (9, 4000, 8500), (15, 70, 20001), (31, 17000, 300), (20, 4100, 9000),
    # rows shorter than a load and than a tile's part of K
    (40, 50, 1), (70, 33, 15), (33, 40, 17), (3, 70, 1), (20, 5, 255), (32, 33, 257),
    # K in slices; tiles of every size, in one round of workgroups and in several
    (40, 100, 50000), (300, 300, 20000), (130, 9000, 256), (500, 1500, 1030), (1300, 5200, 144), (2300, 5000, 257),
    (4100, 6200, 130), (2000, 1999, 4112), (2990, 4001, 2065), (3950, 3901, 2064), (5000, 4100, 1040),
    # whole rounds of one tile and the columns left over on another, in one piece and in slices of K
    (1294, 11946, 1733), (2009, 8627, 1177), (358, 11183, 8230), (381, 11070, 7872)])
def test_product_of_every_variant(gpu_runtime, m, n, k, dtype):
    a, w = _whole(m + k, (m, k)), _whole(n + k, (n, k), -128)
    sa, sw = oracle.uniform(1, (m,), 0.001, 0.03), oracle.uniform(2, (n,), -0.001, 0.001)
    _check_product(_product(gpu_runtime, a, w, sa, sw, dtype), a, w, sa, sw, dtype)


@pytest.mark.parametrize("m,n", [(70000, 40), (70000, 5), (5, 70000)])
def test_product_of_operands_past_4_gib(gpu_runtime, m, n):
    """The last rows of an operand of 4.27e9 bytes (what lies before them is not looked at)."""
    k, last = 61000, 40
    rt, big, small = gpu_runtime, max(m, n), min(m, n)
    tail, other = _whole(1, (last, k)), _whole(2, (small, k))
    scale = oracle.uniform(3, (big,), 0.001, 0.002)
    one = oracle.uniform(4, (small,), 0.001, 0.002)
    out = np.zeros((m, n), np.float32)
    with Device(rt) as dev:
        wide = rt.alloc(big * k)
        dev.held.append(wide)
        rt.upload(wide + (big - last) * k, tail)
        do, narrow, sb, ss = dev.up(out), dev.up(other), dev.up(scale), dev.up(one)
        if m > n:
            rt.gemm_int8_device(wide, narrow, sb, ss, do, m, n, k, F32)
        else:
            rt.gemm_int8_device(narrow, wide, ss, sb, do, m, n, k, F32)
        out = dev.down(out, do)
    if m > n:
        _check_product(out[-last:], tail, other, scale[-last:], one, F32)
    else:
        _check_product(out[:, -last:], other, tail, one, scale[-last:], F32)


@pytest.mark.parametrize("m,n,k", [(2, (1 << 28) + 37, 3), (1, 1 << 30, 1), (1 << 30, 1, 3)])
def test_product_of_very_long_sides(gpu_runtime, m, n, k):
    """More columns than one launch of the kernel for few rows takes, and the most columns and rows: the last ones, and
    those where a launch ends (what lies elsewhere is not looked at)."""
    rt, long, short, span = gpu_runtime, max(m, n), min(m, n), 64
    edges = [at for at in (0, (1 << 27) - 32, (1 << 28) - 32) if at + 2 * span <= long] + [long - span]
    tail, other = _whole(1, (span, k)), _whole(2, (short, k))
    scale, one = oracle.uniform(3, (span,), 0.001, 0.002), oracle.uniform(4, (short,), 0.001, 0.002)
    with Device(rt) as dev:
        wide, scales, out = rt.alloc(long * k), rt.alloc(long * 4), rt.alloc(m * n * 2)
        dev.held += [wide, scales, out]
        for at in edges:
            rt.upload(wide + at * k, tail)
            rt.upload(scales + at * 4, scale)
        narrow, ones = dev.up(other), dev.up(one)
        if m > n:
            rt.gemm_int8_device(wide, narrow, scales, ones, out, m, n, k, BF16)
        else:
            rt.gemm_int8_device(narrow, wide, ones, scales, out, m, n, k, BF16)
        rt.synchronize()
        for at in edges:
            if m > n:
                got = _values(rt.download(np.empty((span, n), np.uint16), out + at * n * 2), BF16)
                _check_product(got, tail, other, scale, one, BF16)
            else:
                got = [rt.download(np.empty(span, np.uint16), out + (row * n + at) * 2) for row in range(m)]
                _check_product(_values(np.stack(got), BF16), other, tail, one, scale, BF16)


# ------------------------------------------------------------------ the cache
class Case:
    """A paged cache on the host and on the device, with the rows that a call brings."""

    def __init__(self, dim, heads, lengths, new, dtype, seed=1, spare=3, extra_rows=0, stride_extra=0, empty=0):
        rng = np.random.default_rng(seed)
        self.dim, self.heads, self.dtype = dim, heads, dtype
        self.lengths = np.array(lengths, np.int32)
        self.new = np.array(new, np.int32)
        counts = [max(0, -(-int(n) // oq.PAGE)) for n in lengths]
        self.pages = sum(counts) + spare
        self.stride = max(counts + [1])
        order = rng.permutation(self.pages)
        self.table = np.full((len(lengths), self.stride), -7, np.int32)  # what is not used is no page
        at = 0
        for i, c in enumerate(counts):
            self.table[i, :c] = order[at:at + c]
            at += c
        self.starts = (empty + np.concatenate([[0], np.cumsum(self.new)])).astype(np.int32)
        self.rows = int(self.starts[-1]) + extra_rows
        self.row_stride = heads * dim + stride_extra
        # a pool full of anything: codes, infinities and NaN among the steps
        fill = rng.integers(0, 256, (self.pages, heads, oq.PAGE * dim + 4 * dim), dtype=np.uint8)
        self.cache = oq.Cache(self.pages, heads, dim, fill)
        self.rng = rng

    def history(self, seed):
        """Values of every token of every sequence, in the row type's precision, stored in the host's cache."""
        g = np.random.default_rng(seed)
        self.k, self.v = [], []
        for i, n in enumerate(self.lengths):
            n = max(0, int(n))
            k = _rounded((g.standard_normal((n, self.heads, self.dim)) * (1 + 3 * (np.arange(self.dim) % 37 == 0))).astype(np.float32), self.dtype)
            v = _rounded(g.standard_normal((n, self.heads, self.dim)).astype(np.float32), self.dtype)
            for t in range(n):
                page = self.table[i, t // oq.PAGE]
                if 0 <= page < self.pages:
                    self.cache.store(page, t % oq.PAGE, k[t], v[t])
            self.k.append(oq.kv4_values(*oq.kv4_quantise(k)))
            self.v.append(oq.kv4_values(*oq.kv4_quantise(v)))
        return self

    def handle(self, dev, pool):
        return p.kv4_cache(pool, dev.up(self.table), dev.up(self.lengths), self.dim, self.heads, self.pages,
                           len(self.lengths), self.stride)

    def places(self):
        """(row, sequence, position) of the rows that belong to a sequence."""
        for i, n in enumerate(self.new):
            for j in range(int(n)):
                yield int(self.starts[i]) + j, i, int(max(0, self.lengths[i])) - int(n) + j


CACHE_CASES = [
    # dim, heads, lengths, new rows, more: rows behind the last sequence, before the first, stride
    dict(dim=128, heads=2, lengths=[1], new=[1]),
    dict(dim=64, heads=1, lengths=[64], new=[64]),
    dict(dim=256, heads=3, lengths=[65, 0, 7], new=[3, 0, 7]),
    dict(dim=128, heads=8, lengths=[130, 64, 1, 200], new=[1, 1, 1, 1], stride_extra=77),
    dict(dim=64, heads=5, lengths=[300, 5], new=[129, 9], extra_rows=6, empty=2, stride_extra=1),  # 9 rows, 5 tokens
    dict(dim=256, heads=1, lengths=[70, 128, 63], new=[70, 60, 1], extra_rows=1),
    dict(dim=128, heads=1, lengths=[2] * 150, new=[1, 0, 2] * 50),
    dict(dim=64, heads=1, lengths=[1] * 5000, new=[1] * 5000),
]


def _rows_of(case, seed):
    x = np.random.default_rng(seed).standard_normal((case.rows, case.row_stride)).astype(np.float32)
    x[:, :case.heads * case.dim] *= np.exp2(np.random.default_rng(seed + 1).integers(-8, 9, (case.rows, 1))).astype(np.float32)
    return _rounded(x, case.dtype)


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("index", range(len(CACHE_CASES)))
def test_cache_pages_and_read_back(gpu_runtime, index, dtype):
    case = Case(dtype=dtype, **CACHE_CASES[index])
    k, v = _rows_of(case, 10), _rows_of(case, 20)
    width = case.heads * case.dim
    shape = (case.heads, case.dim)
    expect_k, expect_v = k.copy(), v.copy()
    expect_k[:], expect_v[:] = -3.0, -4.0  # what a read leaves alone
    written = np.zeros(k.shape, bool)
    for row, seq, pos in case.places():
        if pos < 0:
            continue
        kk, vv = k[row, :width].reshape(shape), v[row, :width].reshape(shape)
        case.cache.store(case.table[seq, pos // oq.PAGE], pos % oq.PAGE, kk, vv)
        written[row, :width] = True
        expect_k[row, :width] = oq.kv4_values(*oq.kv4_quantise(kk)).reshape(-1)
        expect_v[row, :width] = oq.kv4_values(*oq.kv4_quantise(vv)).reshape(-1)
    start = Case(dtype=dtype, **CACHE_CASES[index]).cache.pool
    with Device(gpu_runtime) as dev:
        pool = dev.up(start)
        handle = case.handle(dev, pool)
        starts = dev.up(case.starts)
        lead = 2 if dtype == BF16 else 4
        gpu_runtime.kv4_write_device(handle, dev.up(_bits(k, dtype), lead), dev.up(_bits(v, dtype)), starts, case.rows,
                                     case.row_stride, dtype)
        out = _bits(np.full_like(k, -3.0), dtype)
        other = _bits(np.full_like(v, -4.0), dtype)
        dk, dv = dev.up(out), dev.up(other, lead)
        gpu_runtime.kv4_read_device(handle, dk, dv, starts, case.rows, case.row_stride, dtype)
        got_pool = dev.down(start, pool)
        got_k, got_v = _values(dev.down(out, dk), dtype), _values(dev.down(other, dv), dtype)
        # one of the two alone
        only = dev.up(out)
        gpu_runtime.kv4_read_device(handle, None, only, starts, case.rows, case.row_stride, dtype)
        alone = _values(dev.down(out, only), dtype)
    assert np.array_equal(got_pool, case.cache.pool)
    assert np.array_equal(got_k, expect_k) and np.array_equal(got_v, expect_v)
    expect_v[~written] = -3.0
    assert np.array_equal(alone, expect_v)


def test_cache_groups_of_special_values(gpu_runtime):
    """Ties, zeros, the smallest and largest numbers, infinities and NaN, a group each."""
    case = Case(dim=256, heads=1, lengths=[5], new=[5], dtype=F32)
    x = np.zeros((5, 256), np.float32)
    x[0, :9] = [6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.0]
    x[0, 64:128] = np.float32(1e-45)
    x[0, 128:192] = np.float32(2.0 ** -149) * np.arange(64) * 300000
    x[0, 192:] = np.linspace(-3.4e38, 3.4e38, 64)
    x[1, 3] = np.inf
    x[1, 70] = np.nan
    x[1, 130] = -np.inf
    x[1, 200:] = np.float32(2.0 ** -126) * np.linspace(-1, 1, 56)
    x[2] = -np.abs(np.random.default_rng(3).standard_normal(256))
    x[3] = -0.0
    x[4] = np.exp2(np.random.default_rng(4).uniform(-30, 30, 256))
    with Device(gpu_runtime) as dev:
        pool = dev.up(case.cache.pool)
        handle, starts = case.handle(dev, pool), dev.up(case.starts)
        gpu_runtime.kv4_write_device(handle, dev.up(x), dev.up(-x), starts, 5, 256, F32)
        k, v = np.empty_like(x), np.empty_like(x)
        dk, dv = dev.up(k), dev.up(v)
        gpu_runtime.kv4_read_device(handle, dk, dv, starts, 5, 256, F32)
        k, v = dev.down(k, dk), dev.down(v, dv)
    with np.errstate(over="ignore"):  # 6 s of the largest group lies past fp32's range
        expect = oq.kv4_values(*oq.kv4_quantise(x)).astype(np.float32)
    assert np.isinf(expect).any()
    assert np.array_equal(np.isnan(k), np.isnan(expect)) and np.isnan(k).sum() == 3 * 64
    assert np.array_equal(k, expect, equal_nan=True) and np.array_equal(v, -expect, equal_nan=True)


@pytest.mark.parametrize("power", (-125, -100, -81, 0, 79, 82, 120))
def test_cache_groups_next_to_where_rounding_changes(gpu_runtime, power):
    """Values within two ulps of the middle between two codes, tops within two of where the step changes, and
    zeros of both signs: the page's bits."""
    case = Case(dim=64, heads=2, lengths=[200], new=[200], dtype=F32)
    rng = np.random.default_rng(power + 300)
    x = np.zeros((400, 64), np.float32)
    top = (rng.uniform(1, 2, 400) * 2.0 ** power).astype(np.float32)
    # a step of six bits, six times over: the next top's step is the next
    top[:200] = _beside((6.0 * (32 + np.arange(40) % 32) / 32 * 2.0 ** power).astype(np.float32)).reshape(-1)
    t = (top / np.float32(6.0)).astype(np.float32)
    step = ((t.view(np.uint32) + np.uint32(0x3FFFF)) & np.uint32(0xFFFC0000)).view(np.float32)
    middles = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32)
    x[:, :35] = _beside(step[:, None] * middles).reshape(400, -1) * rng.choice([-1, 1], (400, 35))
    x = np.where(np.abs(x) > top[:, None], np.float32(0.0), x)
    x[:, 40], x[:, 41], x[:, 63] = -0.0, 0.0, top
    x = x.reshape(200, 128)
    k, v = x.reshape(200, 2, 64), -x.reshape(200, 2, 64)
    before = case.cache.pool.copy()
    for row, seq, pos in case.places():
        case.cache.store(case.table[seq, pos // oq.PAGE], pos % oq.PAGE, k[row], v[row])
    with Device(gpu_runtime) as dev:
        pool = dev.up(before)
        handle, starts = case.handle(dev, pool), dev.up(case.starts)
        gpu_runtime.kv4_write_device(handle, dev.up(x), dev.up(-x), starts, 200, 128, F32)
        got = dev.down(before, pool)
    assert np.array_equal(got, case.cache.pool)


def test_cache_past_4_gib_of_pages_and_rows(gpu_runtime):
    """Pages at the end of a pool of 4.6e9 bytes, rows 2^24 - 1 elements apart: written, read back, attended to."""
    rt, dim, heads, group, pages, stride, rows = gpu_runtime, 256, 8, 2, 33000, (1 << 24) - 1, 260
    case = Case(dim, heads, [260, 3], [258, 2], BF16, seed=2)
    case.table[0], case.table[1, 0] = pages - 2 - np.arange(case.stride), pages - 1
    case.pages = pages
    k, v = (_rounded(oracle.normal(s, (rows, heads, dim)), BF16) for s in (1, 2))
    q = _rounded(oracle.normal(3, (rows, heads * group, dim)), BF16)
    block = heads * (oq.PAGE * dim + 4 * dim)
    last = np.zeros((8, block), np.uint8)
    with Device(rt) as dev:
        pool = rt.alloc(pages * block)
        dev.held.append(pool)
        rt.upload(pool + (pages - 8) * block, last)
        wide = rt.alloc(rows * stride * 2)
        dev.held.append(wide)
        q_at, k_at, v_at, o_at = 0, 8192, 16384, 24576  # elements of a row
        for r in range(rows):
            for at, x in ((q_at, q), (k_at, k), (v_at, v)):
                rt.upload(wide + 2 * (r * stride + at), _bits(x[r], BF16))
        handle, starts = case.handle(dev, pool), dev.up(case.starts)
        rt.kv4_write_device(handle, wide + 2 * k_at, wide + 2 * v_at, starts, rows, stride, BF16)
        back = k_at + heads * dim
        rt.kv4_read_device(handle, wide + 2 * back, None, starts, rows, stride, BF16)
        rt.attention_kv4_device(handle, wide, wide + 2 * o_at, starts, rows, heads * group, stride, stride, 258, 260, 0,
                                dim ** -0.5, BF16)
        rt.synchronize()
        read, out = np.zeros_like(_bits(k, BF16)), np.zeros_like(_bits(q, BF16))
        for r in range(rows):
            rt.download(read[r], wide + 2 * (r * stride + back))
            rt.download(out[r], wide + 2 * (r * stride + o_at))
        last = rt.download(last, pool + (pages - 8) * block)
    assert np.array_equal(_values(read, BF16), oq.kv4_values(*oq.kv4_quantise(k)))
    # the two tokens before the call's in sequence 0 and the one in sequence 1: zeros in the pool
    case.k, case.v = [], []
    for i in range(2):
        first, n, old = int(case.starts[i]), int(case.new[i]), int(case.lengths[i] - case.new[i])
        for held, x in ((case.k, k), (case.v, v)):
            held.append(np.concatenate([np.zeros((old, heads, dim)), oq.kv4_values(*oq.kv4_quantise(x[first:first + n]))]))
    _check_attention(_values(out, BF16), case, q, group, BF16)


def test_bad_pages_are_not_written_and_read_back_as_nan(gpu_runtime):
    case = Case(dim=128, heads=2, lengths=[200, 100], new=[200, 100], dtype=F32)
    case.table[0, 1], case.table[0, 2], case.table[1, 0] = case.pages, -1, 0x7FFFFFFF
    case.stride = 3  # tokens 192.. of sequence 0 lie past its table's row
    case.table = np.ascontiguousarray(case.table[:, :3])
    before = case.cache.pool.copy()
    k = _rows_of(case, 5)
    good = np.zeros(case.rows, bool)
    for row, seq, pos in case.places():
        place = pos // oq.PAGE
        good[row] = place < 3 and 0 <= case.table[seq, place] < case.pages
        if good[row]:
            kk = k[row].reshape(2, 128)
            case.cache.store(case.table[seq, place], pos % oq.PAGE, kk, kk)
    with Device(gpu_runtime) as dev:
        pool = dev.up(before)
        handle, starts = case.handle(dev, pool), dev.up(case.starts)
        dk = dev.up(k)
        gpu_runtime.kv4_write_device(handle, dk, dk, starts, case.rows, 256, F32)
        out = np.zeros_like(k)
        do = dev.up(out)
        gpu_runtime.kv4_read_device(handle, do, None, starts, case.rows, 256, F32)
        out, pool = dev.down(out, do), dev.down(before, pool)
    assert good.any() and not good.all()
    assert np.array_equal(pool, case.cache.pool)
    assert np.isnan(out[~good]).all() and np.isfinite(out[good]).all()


# ------------------------------------------------------------------ attention
def _attend(rt, case, q, group, dtype, window=0, scale=None, max_rows=None, max_length=None, pad=0, lead=0):
    """Rows [rows, q_heads, D] of the kernel's output; rows that it leaves alone keep 9."""
    heads = case.heads * group
    width = heads * case.dim
    wide = np.full((case.rows, width + pad), 9.0, np.float32)
    wide[:, :width] = q.reshape(case.rows, width)
    with Device(rt) as dev:
        handle = case.handle(dev, dev.up(case.cache.pool))
        out = _bits(np.full_like(wide, 9.0), dtype)
        do = dev.up(out, lead)
        most = max(1, int(case.new.max())) if max_rows is None else max_rows
        longest = max(1, int(case.lengths.max())) if max_length is None else max_length
        rt.attention_kv4_device(handle, dev.up(_bits(wide, dtype), lead), do, dev.up(case.starts), case.rows, heads,
                                width + pad, width + pad, most, longest, window,
                                case.dim ** -0.5 if scale is None else scale, dtype)
        out = _values(dev.down(out, do), dtype)
    assert np.all(out[:, width:] == 9.0)
    return out[:, :width].reshape(case.rows, heads, case.dim)


def _check_attention(got, case, q, group, dtype, window=0, scale=None):
    scale = case.dim ** -0.5 if scale is None else scale
    scale = float(np.float32(scale))
    mine = np.zeros(case.rows, bool)
    worst = 0.0
    for row, seq, pos in case.places():
        mine[row] = True
        ref, size, reach = oq.attention(q[row].astype(np.float64), case.k[seq], case.v[seq], pos, scale, window)
        tokens = max(1, pos + 1)
        rel = 2 * (case.dim + 16) * 2.0 ** -24 * (1 + reach[:, None]) + 2.0 ** -21 + (tokens / 16 + 64) * 2.0 ** -24
        tol = (rel + (2.0 ** -8 if dtype == BF16 else 0.0)) * size
        tol += (2.0 ** -8 if dtype == BF16 else 2.0 ** -24) * np.abs(ref) + 1e-37
        err = np.abs(got[row].astype(np.float64) - ref)
        assert np.all(np.isfinite(got[row])), (row, seq, pos)
        worst = max(worst, float((err / tol).max()))
        assert np.all(err <= tol), (row, seq, pos, float((err / tol).max()))
    assert np.all(got[~mine] == 9.0)
    print(f"largest error {worst:.3f} of the tolerance", flush=True)


ATTENTION_CASES = [
    # dim, heads, group, lengths, new rows, window
    (128, 2, 4, [1], [1], 0),
    (64, 1, 1, [2, 63, 64, 65], [1, 1, 1, 1], 0),
    (256, 1, 8, [777], [1], 0),
    (128, 8, 4, [300, 1, 0, 129, 1000], [1, 1, 0, 1, 1], 0),
    (128, 1, 16, [640], [1], 0),
    (64, 3, 5, [70, 200], [7, 3], 0),
    (128, 2, 3, [33], [33], 0),
    (256, 2, 2, [150, 64], [100, 64], 0),
    (128, 1, 4, [500, 40], [130, 1], 0),
    (64, 2, 8, [900], [1], 100),
    (128, 2, 2, [400, 90], [70, 90], 33),
    (256, 1, 4, [330], [20], 64),
    (128, 1, 1, [5, 3], [9, 3], 0),  # nine rows of a sequence of five tokens: four see nothing
    (64, 1, 17, [257], [40], 1),     # every row sees its own token alone
    (64, 1, 40, [130], [2], 0),
    (128, 1, 2, [3000], [1], 0),
    (128, 1, 2, [700, 650], [600, 300], 0),
    (64, 2, 4, [600, 70, 300], [500, 1, 120], 0),  # prompts of several tiles beside a single row
    (256, 1, 3, [400, 260], [390, 30], 0),
    (64, 1, 1, [700, 300], [650, 300], 90),
    (128, 3, 8, [100, 20, 5], [90, 20, 30], 0),  # thirty rows of a sequence of five tokens
]


# A max_length that is far too large makes the call look like work for the prompts' kernel, which
# then takes every sequence of more than 64 pairs.
LOOKS_LONG = 1 << 24


@pytest.mark.parametrize("longest", (None, LOOKS_LONG))
@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("index", range(len(ATTENTION_CASES)))
def test_attention_equals_the_definition(gpu_runtime, index, dtype, longest):
    dim, heads, group, lengths, new, window = ATTENTION_CASES[index]
    case = Case(dim, heads, lengths, new, dtype, seed=index, extra_rows=index % 3, empty=index % 2).history(index + 50)
    q = _rounded(oracle.normal(index + 7, (case.rows, heads * group, dim), 0.0, 1.5), dtype)
    got = _attend(gpu_runtime, case, q, group, dtype, window, pad=index % 4 * 3, lead=(index % 2) * 4,
                  max_length=longest)
    _check_attention(got, case, q, group, dtype, window)


@pytest.mark.parametrize("longest", (None, LOOKS_LONG))
@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("dim,lengths,new,first,rows,window", [
    (128, [100, 70], [8, 15], 0, 12, 0),          # the last sequence's rows end behind the call's
    (64, [400, 600], [10, 490], 3, 250, 0),       # and its first sequence's begin before them
    (256, [90, 2000, 40], [2, 1, 9], 1, 4, 0),
    (64, [300, 900], [130, 500], 90, 440, 50)])
def test_rows_that_a_call_has_not_all_of(gpu_runtime, dim, lengths, new, first, rows, window, dtype, longest):
    """Row starts below 0 and past `rows`: the positions of the rows that the call has do not depend on that, for
    writing and reading as for attention."""
    case = Case(dim, 2, lengths, new, dtype, seed=31).history(90)
    case.starts, case.rows = case.starts - first, rows
    assert case.starts[0] <= 0 and case.starts[-1] > rows
    all_places = list(case.places())
    places = [x for x in all_places if 0 <= x[0] < rows]
    case.places = lambda: iter(places)
    # the rows' keys and values are other ones than the cache holds there
    k, v = _rows_of(case, 41), _rows_of(case, 42)
    before = case.cache.pool.copy()
    for row, seq, pos in places:
        kk, vv = k[row].reshape(2, dim), v[row].reshape(2, dim)
        case.cache.store(case.table[seq, pos // oq.PAGE], pos % oq.PAGE, kk, vv)
        case.k[seq][pos], case.v[seq][pos] = (oq.kv4_values(*oq.kv4_quantise(x)) for x in (kk, vv))
    with Device(gpu_runtime) as dev:
        pool = dev.up(before)
        handle, starts = case.handle(dev, pool), dev.up(case.starts)
        gpu_runtime.kv4_write_device(handle, dev.up(_bits(k, dtype)), dev.up(_bits(v, dtype)), starts, rows, 2 * dim, dtype)
        out = _bits(np.zeros_like(k), dtype)
        do = dev.up(out)
        gpu_runtime.kv4_read_device(handle, do, None, starts, rows, 2 * dim, dtype)
        got_pool, read = dev.down(before, pool), _values(dev.down(out, do), dtype)
    assert np.array_equal(got_pool, case.cache.pool)
    for row, seq, pos in places:
        assert np.array_equal(read[row], case.k[seq][pos].reshape(-1)), row
    q = _rounded(oracle.normal(43, (rows, 8, dim)), dtype)
    got = _attend(gpu_runtime, case, q, 4, dtype, window, max_rows=rows if longest else min(rows, max(new)), max_length=longest)
    # As _check_attention, but for what underflows: scores are up to hundreds apart here, and where the token that
    # wins holds a 0 the result is what the others leave.  Relative to a running maximum, which the largest may pass
    # by 2^8, factors below 2^-126 count as 0 (a probability's, a step's times it, or the one that sums so far,
    # of probabilities up to 2^8, are scaled with): less than 2^-117 |v| a token, divided by weights of 1 or more.
    for row, seq, pos in places:
        ref, size, reach = oq.attention(q[row].astype(np.float64), case.k[seq], case.v[seq], pos,
                                        float(np.float32(dim ** -0.5)), window)
        rel = 2 * (dim + 16) * 2.0 ** -24 * (1 + reach[:, None]) + 2.0 ** -21 + ((pos + 1) / 16 + 64) * 2.0 ** -24
        tol = (rel + (2.0 ** -8 if dtype == BF16 else 0.0)) * size + (2.0 ** -8 if dtype == BF16 else 2.0 ** -24) * np.abs(ref)
        tol += (pos + 1) * 2.0 ** -117 * max(6.0, np.abs(case.v[seq]).max())
        assert np.all(np.abs(got[row] - ref) <= tol), (row, seq, pos)
    mine = np.isin(np.arange(rows), [x[0] for x in places])
    assert np.all(got[~mine] == 9.0)


@pytest.mark.parametrize("name,dtype,dim,heads,group,lengths,new,window,plan", PLANNED, ids=[c[0] for c in PLANNED])
def test_attention_as_planned(gpu_runtime, name, dtype, dim, heads, group, lengths, new, window, plan):
    """Truthful hints: every split has pages, joins have all of them to add, beside pieces of prompts too."""
    case = Case(dim, heads, lengths, new, dtype, seed=len(name)).history(len(name) + 60)
    q = _rounded(oracle.normal(len(name) + 7, (case.rows, heads * group, dim), 0.0, 1.5), dtype)
    got = _attend(gpu_runtime, case, q, group, dtype, window)
    _check_attention(got, case, q, group, dtype, window)


@pytest.mark.parametrize("dim", (64, 128, 256))
def test_attention_peaked_and_large_scores(gpu_runtime, dim):
    """Scores of hundreds, which one token wins, and a maximum that keeps growing along the sequence."""
    case = Case(dim, 1, [400, 200], [3, 1], F32, seed=4)
    case.history(9)
    q = oracle.normal(3, (case.rows, 2, dim), 0.0, 30.0)
    # the cache's own values along one direction, rising with the position
    for i, n in enumerate(case.lengths):
        k = (np.arange(n)[:, None, None] / 50.0 * q[0, 0] / np.abs(q[0, 0]).max()).astype(np.float32)
        v = np.random.default_rng(i).standard_normal(k.shape).astype(np.float32)
        for t in range(n):
            case.cache.store(case.table[i, t // oq.PAGE], t % oq.PAGE, k[t], v[t])
        case.k[i], case.v[i] = (oq.kv4_values(*oq.kv4_quantise(x)) for x in (k, v))
    got = _attend(gpu_runtime, case, q, 2, F32)
    _check_attention(got, case, q, 2, F32)


def test_attention_does_not_depend_on_the_launch_hints(gpu_runtime):
    """Too small and too large max_rows and max_length: whole results all the same."""
    case = Case(128, 2, [2000, 90, 700], [50, 1, 3], BF16, seed=8, extra_rows=2).history(12)
    q = _rounded(oracle.normal(5, (case.rows, 8, 128)), BF16)
    for most, longest in ((50, 2000), (1, 1), (56, LOOKS_LONG), (3, 0xFFFFFFFF), (56, 64), (17, LOOKS_LONG)):
        got = _attend(gpu_runtime, case, q, 4, BF16, max_rows=most, max_length=longest)
        _check_attention(got, case, q, 4, BF16)


@pytest.mark.parametrize("longest", (None, LOOKS_LONG))
def test_attention_of_many_sequences(gpu_runtime, longest):
    """More sequences than a search step, a workgroup's threads and a row of the grid hold, prompts among them."""
    lengths = [1 + i * 7 % 90 for i in range(700)]
    new = [n if i % 97 == 5 else i % 3 % (n + 1) for i, n in enumerate(lengths)]
    case = Case(64, 1, lengths, new, BF16, seed=13, extra_rows=3, empty=2).history(77)
    q = _rounded(oracle.normal(19, (case.rows, 2, 64)), BF16)
    _check_attention(_attend(gpu_runtime, case, q, 2, BF16, max_length=longest), case, q, 2, BF16)


@pytest.mark.parametrize("longest", (None, LOOKS_LONG))
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (256, F32)])
def test_attention_gives_equal_bits_again(gpu_runtime, dim, dtype, longest):
    case = Case(dim, 2, [900, 333], [300, 1], dtype, seed=14).history(78)
    q = _rounded(oracle.normal(20, (case.rows, 8, dim)), dtype)
    first, second = (_attend(gpu_runtime, case, q, 4, dtype, max_length=longest) for _ in range(2))
    assert np.array_equal(first, second)


@pytest.mark.parametrize("dim", (64, 128, 256))
@pytest.mark.parametrize("longest", (130, LOOKS_LONG))
def test_attention_ignores_what_is_behind_a_sequence(gpu_runtime, longest, dim):
    """The pool behind the last token, and of pages that are not its own, may hold anything: bit for bit the same."""
    outs = []
    for seed in (1, 2):
        case = Case(dim, 2, [77, 130], [70, 1], BF16, seed=3)
        case.cache.pool[:] = np.random.default_rng(seed).integers(0, 256, case.cache.pool.shape, dtype=np.uint8)
        case.history(30)
        q = _rounded(oracle.normal(6, (case.rows, 4, dim)), BF16)
        outs.append(_attend(gpu_runtime, case, q, 2, BF16, max_length=longest))
    assert np.array_equal(outs[0], outs[1]) and np.isfinite(outs[0]).all()


@pytest.mark.parametrize("longest", (200, LOOKS_LONG))
@pytest.mark.parametrize("window", (0, 90))
def test_attention_of_bad_pages_and_values(gpu_runtime, longest, window):
    """A bad page, a place past the table and a NaN key make the rows NaN that see them, and only those."""
    case = Case(64, 1, [200, 70, 66], [140, 70, 2], F32, seed=5).history(31)
    case.table[0, 2] = case.pages
    nan = np.full((1, 64), np.nan, np.float32)
    case.cache.store(case.table[1, 0], 40, nan, np.ones((1, 64), np.float32))
    case.table = np.ascontiguousarray(case.table[:, :3])
    case.stride = 3  # tokens 192.. of sequence 0 have no place
    q = oracle.normal(8, (case.rows, 2, 64))
    got = _attend(gpu_runtime, case, q, 2, F32, window, max_length=longest)
    for row, seq, pos in case.places():
        first = max(0, pos - window + 1) if window else 0
        bad = (seq == 0 and pos >= 128) or (seq == 1 and first <= 40 <= pos)
        assert np.isnan(got[row]).all() if bad else np.isfinite(got[row]).all(), (row, seq, pos)


@pytest.mark.parametrize("longest", (200, LOOKS_LONG))
@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("window", (0, 20))
def test_attention_to_values_that_are_not_finite(gpu_runtime, longest, dtype, window):
    """A NaN or infinite value group reaches its own channels, and only rows that see it."""
    case = Case(128, 1, [200], [100], dtype, seed=6).history(32)
    v = np.ones((1, 128), np.float32)
    v[0, 70] = np.inf
    for at in (20, 150):
        case.cache.store(case.table[0, at // 64], at % 64, np.ones((1, 128), np.float32), v)
    q = _rounded(oracle.normal(9, (case.rows, 1, 128)), dtype)
    got = _attend(gpu_runtime, case, q, 1, dtype, window, max_length=longest)
    for row, seq, pos in case.places():
        first = max(0, pos - window + 1) if window else 0
        assert np.isfinite(got[row, :, :64]).all()
        spoilt = first <= 20 <= pos or first <= 150 <= pos
        assert np.isnan(got[row, :, 64:]).all() if spoilt else np.isfinite(got[row, :, 64:]).all(), pos


# With a window max_length alone does not: a call looks as long as max_rows and the window.  Rows that no sequence
# has make it look like work for the prompts' kernel, if max_rows counts them.
IDLE_ROWS = 8000


@pytest.mark.parametrize("idle", (0, IDLE_ROWS))
@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("window,at", [(0, 150), (0, 199), (20, 105), (20, 150)])
def test_attention_to_values_at_the_end_of_the_range(gpu_runtime, idle, dtype, window, at):
    """Six steps of a group of magnitudes above 2^128 * 63 / 64 are past fp32's range, though the step is not: rows
    that do not see the token (before it, or with a window that has left it behind) are as without it."""
    case = Case(128, 1, [200], [100], dtype, seed=6, extra_rows=idle).history(32)
    v = np.ones((1, 128), np.float32)
    v[0, 64:] = _rounded(np.linspace(-3.385e38, 3.385e38, 64).astype(np.float32), dtype)
    case.cache.store(case.table[0, at // 64], at % 64, np.ones((1, 128), np.float32), v)
    case.k[0][at], case.v[0][at] = 1.0, oq.kv4_values(*oq.kv4_quantise(v))
    assert np.abs(case.v[0][at]).max() > np.finfo(np.float32).max
    q = _rounded(oracle.normal(9, (case.rows, 1, 128)), dtype)
    got = _attend(gpu_runtime, case, q, 1, dtype, window, max_rows=case.rows, max_length=LOOKS_LONG if idle else None)
    sees = np.zeros(case.rows, bool)
    for row, _, pos in case.places():
        sees[row] = at <= pos and (not window or pos - window < at)
    assert np.isfinite(got[:, :, :64]).all() and np.isfinite(got[~sees]).all() and sees.any() and not sees[:100].all()
    case.v[0][at] = 0.0  # what the other rows are held to has it nowhere
    got[sees] = 9.0
    places = [x for x in case.places() if not sees[x[0]]]
    case.places = lambda: iter(places)
    _check_attention(got, case, q, 1, dtype, window)


# ------------------------------------------------------------------ a step of the whole path
@pytest.mark.parametrize("dtype", (F32, BF16))
def test_decode_step(gpu_runtime, dtype):
    """Rows to 8 bits, the projection of queries, keys and values, the cache, attention, and the projection back,
    queued one after the other without a wait, against the same chain from the definitions."""
    rt, heads, group, dim, hidden = gpu_runtime, 2, 4, 128, 640
    q_width, kv_width = heads * group * dim, heads * dim
    width = q_width + 2 * kv_width
    case = Case(dim, heads, [130, 65, 64, 3], [1, 1, 1, 3], dtype, seed=11).history(40)
    x = _rounded(oracle.normal(50, (case.rows, hidden)), dtype)
    w, wo = _whole(51, (width, hidden)), _whole(52, (hidden, q_width))
    sw, so = oracle.uniform(53, (width,), 0.0002, 0.0006), oracle.uniform(54, (hidden,), 0.0002, 0.0006)
    size = 2 if dtype == BF16 else 4
    empty = lambda *shape: _bits(np.zeros(shape, np.float32), dtype)  # noqa: E731
    with Device(rt) as dev:
        handle = case.handle(dev, dev.up(case.cache.pool))
        starts = dev.up(case.starts)
        q8, s8 = np.zeros((case.rows, hidden), np.int8), np.zeros(case.rows, np.float32)
        dq8, ds8 = dev.up(q8), dev.up(s8)
        qkv, attn, back = empty(case.rows, width), empty(case.rows, q_width), empty(case.rows, hidden)
        dqkv, dattn, dback = dev.up(qkv), dev.up(attn), dev.up(back)
        a8, sa8 = np.zeros((case.rows, q_width), np.int8), np.zeros(case.rows, np.float32)
        da8, dsa8 = dev.up(a8), dev.up(sa8)
        rt.quantize_rows_int8_device(dev.up(_bits(x, dtype)), dq8, ds8, case.rows, hidden, hidden, dtype)
        rt.gemm_int8_device(dq8, dev.up(w), ds8, dev.up(sw), dqkv, case.rows, width, hidden, dtype)
        rt.kv4_write_device(handle, dqkv + q_width * size, dqkv + (q_width + kv_width) * size, starts, case.rows, width,
                            dtype)
        rt.attention_kv4_device(handle, dqkv, dattn, starts, case.rows, heads * group, width, q_width, 3, 130, 0,
                                dim ** -0.5, dtype)
        rt.quantize_rows_int8_device(dattn, da8, dsa8, case.rows, q_width, q_width, dtype)
        rt.gemm_int8_device(da8, dev.up(wo), dsa8, dev.up(so), dback, case.rows, hidden, q_width, dtype)
        qkv, attn, back = (_values(dev.down(h, d), dtype) for h, d in ((qkv, dqkv), (attn, dattn), (back, dback)))
        q8, s8, a8, sa8 = dev.down(q8, dq8), dev.down(s8, ds8), dev.down(a8, da8), dev.down(sa8, dsa8)
    # each step against its definition on what the step before gave
    eq8, es8 = oq.quantize_rows(x)
    assert np.array_equal(q8, eq8) and np.array_equal(s8, es8)
    _check_product(qkv, q8, w, s8, sw, dtype)
    for row, seq, pos in case.places():
        for held, at in ((case.k, q_width), (case.v, q_width + kv_width)):
            held[seq][pos] = oq.kv4_values(*oq.kv4_quantise(qkv[row, at:at + kv_width].reshape(heads, dim)))
    _check_attention(attn.reshape(case.rows, heads * group, dim), case, qkv[:, :q_width].reshape(case.rows, heads * group, dim),
                     group, dtype)
    ea8, esa8 = oq.quantize_rows(attn)
    assert np.array_equal(a8, ea8) and np.array_equal(sa8, esa8)
    _check_product(back, a8, wo, sa8, so, dtype)


def _calls(rt, dev, seed, sizes):
    """Queues a product in slices of K, one of padded rows and an attention in splits, of the sizes given, without a
    wait; what checks them."""
    checks = []
    for i, (m, n, k, length) in enumerate(sizes):
        a, w = _whole(seed + i, (m, k)), _whole(seed + i + 9, (n, k))
        sa, sw = oracle.uniform(1, (m,), 0.001, 0.03), oracle.uniform(2, (n,), -0.001, 0.001)
        c = np.zeros((m, n), np.float32)
        dc = dev.up(c)
        rt.gemm_int8_device(dev.up(a), dev.up(w), dev.up(sa), dev.up(sw), dc, m, n, k, F32)
        case = Case(64, 2, [length, 5], [1, 1], F32, seed=seed + i).history(seed + i)
        q = oracle.normal(seed + i, (2, 4, 64))
        out = np.zeros((2, 256), np.float32)
        do = dev.up(out)
        rt.attention_kv4_device(case.handle(dev, dev.up(case.cache.pool)), dev.up(q), do, dev.up(case.starts), 2, 4, 256, 256,
                                1, length, 0, 0.125, F32)

        def check(a=a, w=w, sa=sa, sw=sw, c=c, dc=dc, case=case, q=q, out=out, do=do):
            _check_product(dev.down(c, dc), a, w, sa, sw, F32)
            _check_attention(dev.down(out, do).reshape(2, 4, 64), case, q, 2, F32)
        checks.append(check)
    return checks


def test_calls_that_share_and_grow_the_workspaces(gpu_runtime):
    with Device(gpu_runtime) as dev:
        for check in _calls(gpu_runtime, dev, 60, [(40, 60, 9000, 700), (40, 3000, 4095, 3000), (70, 50, 2001, 100),
                                                   (600, 500, 4112, 1300), (40, 60, 9001, 900)]):
            check()


def test_calls_from_two_threads(gpu_runtime):
    from concurrent.futures import ThreadPoolExecutor

    def run(seed):
        with Device(gpu_runtime) as dev:
            for check in _calls(gpu_runtime, dev, seed, [(33 + seed, 90, 3000 + seed, 400 + seed)] * 6):
                check()
        return True

    with ThreadPoolExecutor(2) as pool:
        assert all(pool.map(run, (1, 2)))


# ------------------------------------------------------------------ bits of the probabilities
@pytest.mark.parametrize("longest", (None, LOOKS_LONG))
@pytest.mark.parametrize("dim", (64, 128, 256))
def test_attention_of_bf16_rows_carries_16_bits_of_the_probabilities(gpu_runtime, dim, longest):
    """With either kernel, so that the launch hints do not choose the precision.  A probability is cut to eight bits and
    the rest, below 2^-7 of it, rounded to eight: off by at most 2^-7 * 2^-8 = 2^-15.  Beside that and what fp32 sums
    add (see above) a result is off by its own rounding alone, half the distance of its neighbours.  Small queries
    keep the fp32 part below 2^-15 (eight-bit probabilities are off by up to 2^-8, about 1e-4 of W here)."""
    case = Case(dim, 1, [260], [200], BF16, seed=21).history(79)
    q = _rounded(oracle.normal(22, (case.rows, 1, dim), 0.0, 0.05), BF16)
    got = _attend(gpu_runtime, case, q, 1, BF16, max_length=longest).astype(np.float64)
    worst = 0.0
    for row, seq, pos in case.places():
        ref, size, reach = oq.attention(q[row].astype(np.float64), case.k[seq], case.v[seq], pos, float(np.float32(dim ** -0.5)))
        rel = 2 * (dim + 16) * 2.0 ** -24 * (1 + reach[:, None]) + 2.0 ** -21 + ((pos + 1) / 16 + 64) * 2.0 ** -24
        off = (rel + 2.0 ** -15) * size
        half = 2.0 ** (np.floor(np.log2(np.abs(ref) + off)) - 8)
        err = np.abs(got[row] - ref)
        worst = max(worst, float((err / (half + off)).max()))
    assert worst <= 1.0, worst
