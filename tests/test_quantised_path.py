"""The quantised decode path without a device: the oracle's definitions, and every refusal of
the entry points.  Refusals are checked on a runtime that has no device, so that nothing is
launched; valid arguments stop there at INIT with the runtime's own detail."""
from __future__ import annotations

import ctypes
from ctypes import byref, c_int, c_uint32

import numpy as np
import pytest

import oracle
from oracle import quantised as oq
from oct_amd import prometheus as p

OK = 1 << 20  # an aligned address; nothing is dereferenced on these paths


@pytest.fixture(scope="module")
def rt():
    runtime = p.NativeRuntime(test_flags=p.TESTCFG_SKIP_VULKAN_INIT)
    yield runtime
    runtime.close()


# ------------------------------------------------------------------ definitions
def test_cache_values_stay_within_a_step():
    x = oracle.normal(3, (500, 128)) * np.exp2(oracle.uniform(4, (500, 1), -60.0, 60.0))
    codes, steps = oq.kv4_quantise(x)
    v = oq.kv4_values(codes, steps)
    step = np.repeat((steps.astype(np.uint32) << 16).view(np.float32), 64, axis=-1)
    assert np.all(np.abs(v - x) <= step * (1 + 1e-6))
    # at most 1/32 above the largest magnitude / 6, and never below it
    top = np.abs(x.reshape(500, 2, 64)).max(-1)
    assert np.all(step[:, ::64] * 6 >= top * (1 - 1e-6)) and np.all(step[:, ::64] * 6 <= top * (1 + 1 / 16))
    # eight significant bits: bf16 holds every value
    assert np.array_equal(oracle.from_bf16(oracle.to_bf16(v.astype(np.float32))).astype(np.float64), v)


def smallest_rows():
    """Rows of whole multiples of 2^-149, whose scales are such multiples too, and by whole numbers what they become:
    the scale is m / 127 rounded to a multiple, x / scale is rounded to fp32 and then to a whole number, which is
    held within 127.  m runs over all that a scale so small can make larger than that, and their neighbours."""
    m = np.arange(1, 17000, dtype=np.int64)
    units = np.stack([m, -m, m - 1, -(m * 2 // 3), m // 2, m * 0 + 1, m * 0, m // 64], -1)
    scale = (2 * m + 127) // 254  # no ties: 127 is odd
    quotient = (units / np.maximum(scale, 1)[:, None]).astype(np.float32).astype(np.float64)
    q = np.where(scale[:, None] > 0, np.clip(np.rint(quotient), -127, 127), 0).astype(np.int64)
    unit = 2.0 ** -149
    return (units * unit).astype(np.float32), q, (scale * unit).astype(np.float32)


def test_rows_of_the_smallest_numbers_keep_their_sign_and_range():
    x, q, scale = smallest_rows()
    got, got_scale = oq.quantize_rows(x)
    assert np.array_equal(got_scale, scale)
    assert np.all(got[x > 0] >= 0) and np.all(got[x < 0] <= 0) and got.min() == -127 and got.max() == 127
    assert np.array_equal(got, q)


# Calls whose sizes are what they say, so that what they are planned as happens: name, type, head width, key heads,
# group, lengths, new rows, window; splits, whether the prompts' kernel runs, sums that a thread of the join adds,
# pages of a split.
PLANNED = [
    ("more splits than parts, 64", p.DTYPE_F32, 64, 1, 2, [5000], [1], 0, (20, 0, 4, 4)),
    ("more splits than parts, 64, bf16", p.DTYPE_BF16, 64, 1, 2, [5000, 1300, 70], [1, 2, 1], 0, (20, 0, 4, 4)),
    ("more splits than parts, 128", p.DTYPE_BF16, 128, 1, 4, [3000], [1], 0, (12, 0, 8, 4)),
    ("more splits than parts, 256", p.DTYPE_F32, 256, 1, 1, [2000], [1], 0, (8, 0, 16, 4)),
    ("the most splits", p.DTYPE_BF16, 256, 1, 8, [16300, 100], [1, 1], 0, (64, 0, 16, 4)),
    ("splits of 16 pages", p.DTYPE_BF16, 64, 8, 1, [2500, 1200] + [10 + 5 * i for i in range(62)], [1] * 64, 0, (3, 0, 1, 16)),
    ("splits of 32 pages", p.DTYPE_BF16, 64, 8, 2, [4200, 3100, 2100] + [9 + 4 * i for i in range(61)], [1] * 64, 0, (3, 0, 1, 32)),
    ("prompts beside splits, 64", p.DTYPE_BF16, 64, 2, 4, [400, 20000, 90], [300, 1, 20], 0, (40, 1, 4, 8)),
    ("prompts beside splits, 128", p.DTYPE_F32, 128, 2, 4, [20000, 500, 3000, 70], [2, 280, 5, 70], 0, (20, 1, 8, 16)),
    ("prompts beside splits, 256", p.DTYPE_BF16, 256, 1, 8, [350, 9600], [330, 1], 0, (38, 1, 16, 4)),
    ("prompts in a window", p.DTYPE_BF16, 64, 3, 4, [2300, 900, 1500], [1500, 600, 1], 200, (8, 1, 1, 4)),
    ("prompts in a narrow window, fp32", p.DTYPE_F32, 128, 3, 4, [1600, 1900], [1600, 500], 70, (8, 1, 1, 4)),
    ("prompts in a wide window", p.DTYPE_BF16, 256, 2, 4, [2400], [1300], 1000, (0, 1, 1, 1)),
]


def test_cache_ties_go_to_the_even_code():
    x = np.zeros((1, 64), np.float32)
    x[0, :9] = [6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.0]  # step 1
    v = oq.kv4_values(*oq.kv4_quantise(x))[0, :9]
    assert v.tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -4.0]


def test_key_order_is_a_permutation_within_groups_of_64():
    for dim in (64, 128, 256):
        order = oq.key_order(dim)
        assert sorted(order) == list(range(dim))
        assert np.array_equal(order[8 * np.arange(dim // 8)] % 8, np.zeros(dim // 8))


def test_page_bytes():
    assert p.kv4_page_bytes(128, 8) == 8 * (64 * 128 + 4 * 128)
    assert p.kv4_page_bytes(64, 1) == 64 * 64 + 256 and p.kv4_page_bytes(256, 1024) == 1024 * 17408
    for dim, heads in ((0, 1), (32, 1), (96, 1), (512, 1), (128, 0), (128, 1025)):
        assert p.kv4_page_bytes(dim, heads) == 0


# ------------------------------------------------------------------ refusals
def _call(rt, name, *args):
    stage, detail = c_uint32(99), c_int(99)
    rc = getattr(rt.lib, name)(rt.handle, *args, byref(stage), byref(detail))
    return rc, stage.value, detail.value


def _refused(result):
    return result == (p.PROM_ERROR, p.STAGE_INIT, p.DETAIL_INVALID_ARGUMENT)


def _no_device(result):
    return result == (p.PROM_ERROR, p.STAGE_INIT, p.DETAIL_HIP_UNAVAILABLE)


ROWS = dict(x=OK, q=OK, s=OK, rows=4, width=64, stride=64, dtype=p.DTYPE_BF16)


def _rows(rt, **change):
    a = dict(ROWS, **change)
    return _call(rt, "prometheus_reactor_runtime_quantize_rows_int8_device", a["x"], a["q"], a["s"], a["rows"],
                 a["width"], a["stride"], a["dtype"])


@pytest.mark.parametrize("change", [dict(x=0), dict(q=0), dict(s=0), dict(rows=0), dict(width=0), dict(stride=63),
                                    dict(dtype=2), dict(x=OK + 1), dict(x=OK + 2, dtype=p.DTYPE_F32), dict(s=OK + 2),
                                    dict(rows=1 << 20, stride=1 << 20)])
def test_quantize_rows_refuses(rt, change):
    assert _refused(_rows(rt, **change)), change


def test_quantize_rows_takes(rt):
    for change in ({}, dict(x=OK + 2, q=OK + 1), dict(stride=65), dict(rows=(1 << 20) - 1, stride=1 << 20)):
        assert _no_device(_rows(rt, **change)), change


PRODUCT = dict(a=OK, w=OK, sa=OK, sw=OK, c=OK, m=3, n=5, k=7, dtype=p.DTYPE_F32)


def _product(rt, **change):
    a = dict(PRODUCT, **change)
    return _call(rt, "prometheus_reactor_runtime_gemm_int8_device", a["a"], a["w"], a["sa"], a["sw"], a["c"], a["m"],
                 a["n"], a["k"], a["dtype"])


def test_int8_product_refuses_in_the_order_of_the_other_products(rt):
    for name in ("a", "w", "sa", "sw", "c"):
        assert _product(rt, **{name: 0, "m": 0}) == (p.PROM_ERROR, p.STAGE_TRANSFER_IN, p.PROM_ERROR)
    for name in ("m", "n", "k"):
        assert _product(rt, **{name: 0}) == (p.PROM_ERROR, p.STAGE_INIT, p.PROM_ERROR)
    for change in (dict(m=1 << 16, n=1 << 16), dict(m=1 << 31), dict(n=1 << 20, k=1 << 12)):
        assert _product(rt, **change) == (p.PROM_ERROR, p.STAGE_TRANSFER_IN, p.DETAIL_SIZE_OVERFLOW), change
    for change in (dict(k=p.GEMM_INT8_MAX_K + 1), dict(dtype=2), dict(sa=OK + 2), dict(sw=OK + 1), dict(c=OK + 2),
                   dict(c=OK + 1, dtype=p.DTYPE_BF16)):
        assert _refused(_product(rt, **change)), change
    for change in ({}, dict(k=p.GEMM_INT8_MAX_K), dict(a=OK + 1, w=OK + 3), dict(c=OK + 2, dtype=p.DTYPE_BF16)):
        assert _no_device(_product(rt, **change)), change


def test_int8_product_refuses_sides_past_its_counting(rt):
    side = p.GEMM_INT8_MAX_SIDE
    for change in (dict(m=side + 1, n=1, k=1), dict(m=1, n=side + 1, k=1), dict(m=1, n=0x7FFFFFFF, k=1)):
        assert _product(rt, **change) == (p.PROM_ERROR, p.STAGE_TRANSFER_IN, p.DETAIL_SIZE_OVERFLOW), change
    for change in (dict(m=side, n=1, k=1), dict(m=3, n=side, k=1)):
        assert _no_device(_product(rt, **change)), change


CACHE = dict(head_dim=128, kv_heads=2, pages=5, sequences=3, table_stride=4, pool=OK, page_table=OK, lengths=OK)
BAD_CACHES = [dict(struct_size=8), dict(head_dim=96), dict(head_dim=0), dict(kv_heads=0), dict(kv_heads=1025),
              dict(pages=0), dict(pages=1 << 31), dict(sequences=0), dict(sequences=(1 << 20) + 1),
              dict(sequences=1 << 20, kv_heads=5), dict(table_stride=0), dict(table_stride=(1 << 24) + 1), dict(pool=0),
              dict(pool=OK + 8), dict(page_table=0), dict(page_table=OK + 2), dict(lengths=0), dict(lengths=OK + 1)]


def _struct(cls, values):
    s = cls()
    s.struct_size = ctypes.sizeof(cls)
    for name, value in values.items():
        setattr(s, name, value)
    return s


def _cache_call(rt, name, cls, cache, request):
    c = None if cache is None else byref(_struct(p.PrometheusKv4Cache, cache))
    r = None if request is None else byref(_struct(cls, request))
    return _call(rt, name, c, r)


CACHE_ROWS = dict(dtype=p.DTYPE_F32, rows=6, row_stride=256, k=OK, v=OK, row_starts=OK)


def _cache_rows(rt, write, cache=CACHE, request=CACHE_ROWS):
    name = "prometheus_reactor_runtime_kv4_%s_device" % ("write" if write else "read")
    return _cache_call(rt, name, p.PrometheusKv4RowsRequest, cache, request)


@pytest.mark.parametrize("write", (True, False))
def test_cache_rows_refuse(rt, write):
    assert _refused(_cache_rows(rt, write, cache=None)) and _refused(_cache_rows(rt, write, request=None))
    for change in BAD_CACHES:
        assert _refused(_cache_rows(rt, write, cache=dict(CACHE, **change))), change
    for change in (dict(struct_size=4), dict(dtype=2), dict(rows=0), dict(rows=(1 << 22) + 1), dict(row_stride=255),
                   dict(row_stride=1 << 24), dict(k=OK + 2), dict(v=OK + 1), dict(k=0, v=0), dict(row_starts=0),
                   dict(row_starts=OK + 2)):
        assert _refused(_cache_rows(rt, write, request=dict(CACHE_ROWS, **change))), change
    for change in (dict(k=0), dict(v=0)):
        result = _cache_rows(rt, write, request=dict(CACHE_ROWS, **change))
        assert _refused(result) if write else _no_device(result), change
    assert _no_device(_cache_rows(rt, write))
    assert _no_device(_cache_rows(rt, write, request=dict(CACHE_ROWS, dtype=p.DTYPE_BF16, k=OK + 2, v=OK + 6)))


ATTENTION = dict(dtype=p.DTYPE_BF16, rows=6, q_heads=8, q_stride=1024, out_stride=1024, max_rows=4, max_length=200,
                 window=0, scale=0.1, q=OK, out=OK, row_starts=OK)


def _attention(rt, cache=CACHE, request=ATTENTION):
    return _cache_call(rt, "prometheus_reactor_runtime_attention_kv4_device", p.PrometheusKv4AttentionRequest, cache,
                       request)


def test_attention_refuses(rt):
    assert _refused(_attention(rt, cache=None)) and _refused(_attention(rt, request=None))
    for change in BAD_CACHES:
        assert _refused(_attention(rt, cache=dict(CACHE, **change))), change
    for change in (dict(struct_size=4), dict(dtype=2), dict(rows=0), dict(rows=(1 << 22) + 1), dict(q_heads=0),
                   dict(q_heads=7), dict(q_heads=(1 << 16) + 2), dict(rows=1 << 17, q_heads=1 << 15, q_stride=1 << 22, out_stride=1 << 22),
                   dict(q_stride=1023), dict(q_stride=1 << 24),
                   dict(out_stride=1023), dict(out_stride=1 << 24), dict(max_rows=0), dict(max_rows=7),
                   dict(max_length=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")),
                   dict(scale=float("nan")), dict(q=0), dict(q=OK + 1), dict(out=0), dict(out=OK + 1),
                   dict(row_starts=0), dict(row_starts=OK + 2), dict(dtype=p.DTYPE_F32, q=OK + 2)):
        assert _refused(_attention(rt, request=dict(ATTENTION, **change))), change
    assert _no_device(_attention(rt))
    assert _no_device(_attention(rt, request=dict(ATTENTION, window=1, max_length=0xFFFFFFFF, q=OK + 2, out=OK + 6)))


def test_attention_refuses_scales_past_the_range_in_base_2(rt):
    """The softmax is in base 2: scale * log2(e) has to be finite too, or equal scores would give NaN."""
    most = np.float32(2.0 ** 128 / np.log2(np.e) * (1 - 2.0 ** -22))
    for scale in (np.finfo(np.float32).max, np.float32(2.4e38), np.float32(2.0 ** 128 / np.log2(np.e) * (1 + 2.0 ** -22))):
        assert np.isfinite(scale) and _refused(_attention(rt, request=dict(ATTENTION, scale=float(scale)))), scale
    for scale in (most, np.float32(1e-45)):
        assert _no_device(_attention(rt, request=dict(ATTENTION, scale=float(scale)))), scale


def test_unknown_handles_are_refused(rt):
    stage, detail = c_uint32(99), c_int(99)
    lib = rt.lib
    calls = [
        lambda: lib.prometheus_reactor_runtime_quantize_rows_int8_device(OK, OK, OK, OK, 1, 1, 1, 0, byref(stage), byref(detail)),
        lambda: lib.prometheus_reactor_runtime_gemm_int8_device(OK, OK, OK, OK, OK, OK, 1, 1, 1, 0, byref(stage), byref(detail)),
        lambda: lib.prometheus_reactor_runtime_kv4_write_device(OK, None, None, byref(stage), byref(detail)),
        lambda: lib.prometheus_reactor_runtime_kv4_read_device(None, None, None, byref(stage), byref(detail)),
        lambda: lib.prometheus_reactor_runtime_attention_kv4_device(OK, None, None, None, None),
    ]
    for call in calls:
        stage.value = detail.value = 99
        assert call() == p.PROM_INVALID_HANDLE
    # the wrappers raise what the library refuses
    with pytest.raises(p.ReactorIssue):
        rt.quantize_rows_int8_device(0, OK, OK, 1, 1, 1, p.DTYPE_F32)
    with pytest.raises(p.ReactorIssue):
        rt.attention_kv4_device(p.kv4_cache(0, OK, OK, 128, 1, 1, 1, 1), OK, OK, OK, 1, 1, 128, 128, 1, 1, 0, 1.0,
                                p.DTYPE_F32)


def test_struct_layouts_match_the_header(tmp_path):
    import subprocess
    from pathlib import Path

    header = Path(p.PACKAGE_DIR).parent / "include" / "prometheus_reactor.h"
    classes = (p.PrometheusKv4Cache, p.PrometheusKv4RowsRequest, p.PrometheusKv4AttentionRequest)
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void){"]
    expect = []
    for cls in classes:
        lines.append(f'printf("%zu\\n", sizeof({cls.__name__}));')
        expect.append(ctypes.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({cls.__name__}, {field}));')
            expect.append(getattr(cls, field).offset)
    lines.append(f'printf("%u %u %u %u\\n", PROM_GEMM_INT8_MAX_K, PROM_KV4_PAGE_TOKENS, PROM_DTYPE_BF16, PROM_DETAIL_PATH_HIP_MFMA_INT8);')
    (tmp_path / "l.c").write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(tmp_path / "l"), str(tmp_path / "l.c")], check=True)
    out = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in out] == expect + [p.GEMM_INT8_MAX_K, p.KV4_PAGE_TOKENS, p.DTYPE_BF16,
                                              p.DETAIL_PATH_HIP_MFMA_INT8]
