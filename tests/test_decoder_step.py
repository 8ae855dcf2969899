"""The rest of a decoder's step without a device: the oracle's definitions, and every refusal of the entry points.
Refusals are checked on a runtime that has no device, so that nothing is launched; valid arguments stop there at INIT
with the runtime's own detail."""
from __future__ import annotations

import ctypes
import math
import subprocess
from ctypes import byref, c_int, c_uint32
from pathlib import Path

import numpy as np
import pytest

import oracle
from oracle import decoder_step as od
from oracle import quantised as oq
from oct_amd import prometheus as p

OK = 1 << 20  # an aligned address; nothing is dereferenced on these paths
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def rt():
    runtime = p.NativeRuntime(test_flags=p.TESTCFG_SKIP_VULKAN_INIT)
    yield runtime
    runtime.close()


# ------------------------------------------------------------------ definitions
def test_a_group_of_64_is_the_caches_group():
    w = oracle.normal(5, (40, 192)) * np.exp2(oracle.uniform(6, (40, 1), -40.0, 40.0))
    codes, steps = od.w4_quantise(w, 64)
    kv_codes, kv_steps = oq.kv4_quantise(w)
    assert np.array_equal(steps, kv_steps) and np.array_equal(codes, kv_codes)
    assert np.array_equal(od.w4_values(codes, steps, 64), oq.kv4_values(kv_codes, kv_steps))


@pytest.mark.parametrize("group", (32, 64, 128))
def test_weights_stay_within_a_step(group):
    w = oracle.normal(3, (30, 300)) * np.exp2(oracle.uniform(4, (30, 1), -60.0, 60.0))
    codes, steps = od.w4_quantise(w, group)
    v = od.w4_values(codes, steps, group)
    step = np.repeat((steps.astype(np.uint32) << 16).view(np.float32), group, axis=-1)[:, :300]
    assert np.all(np.abs(v - w) <= step * (1 + 1e-6))
    assert np.array_equal(oracle.from_bf16(oracle.to_bf16(v.astype(np.float32))).astype(np.float64), v)


def test_packed_bytes():
    """Each code and step is somewhere, once, and nothing else is."""
    for n, k, group in ((1, 1, 32), (16, 128, 128), (17, 129, 64), (33, 300, 32)):
        codes = np.random.default_rng(n).integers(1, 16, (n, k)).astype(np.uint8)
        steps = np.random.default_rng(k).integers(1, 1 << 15, (n, -(-k // group))).astype(np.uint16)
        packed = od.w4_pack(codes, steps, group)
        assert packed.nbytes == p.w4_bytes(n, k, group)
        tiles = -(-n // 16) * -(-k // 128)
        nibbles = np.stack((packed[:tiles * 1024] & 15, packed[:tiles * 1024] >> 4))
        assert np.array_equal(np.sort(nibbles[nibbles > 0]), np.sort(codes.reshape(-1)))
        held = packed[tiles * 1024:].view(np.uint16)
        assert np.array_equal(np.sort(held[held > 0]), np.sort(steps.reshape(-1)))
    # the first lane's four words of a tile are its row's columns 0, 32, 64 and 96
    codes = np.zeros((16, 128), np.uint8)
    codes[0, [0, 33, 70, 103]] = [1, 2, 3, 4]
    packed = od.w4_pack(codes, np.ones((16, 4), np.uint16), 32)
    assert packed[:16].tolist() == [1, 0, 0, 0, 0x20, 0, 0, 0, 0, 0, 0, 3, 0, 0, 0, 0x40]


def test_w4_bytes():
    assert p.w4_bytes(16, 128, 128) == 1024 + 32 and p.w4_bytes(1, 1, 32) == 1024 + 128
    assert p.w4_bytes(1 << 24, 1 << 20, 64) == (1 << 33) * (1024 + 64)
    for n, k, group in ((0, 1, 32), (1, 0, 32), (1, 1, 0), (1, 1, 16), (1, 1, 96), (1, 1, 256), ((1 << 24) + 1, 1, 32),
                        (1, (1 << 20) + 1, 32)):
        assert p.w4_bytes(n, k, group) == 0


def test_activations():
    g = np.array([-30.0, -3.0, -0.5, 0.0, 0.5, 3.0, 30.0])
    # 1 + tanh is rounded to 2^-53, times |g| / 2 <= 15: 1.7e-15 of absolute error in this form
    assert np.allclose(od.activation(g, False), g * 0.5 * (1 + np.tanh(g / 2)), rtol=1e-9, atol=1e-14)
    gelu = 0.5 * g * (1 + np.tanh(np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)))
    assert np.allclose(od.activation(g, True), gelu, rtol=1e-9, atol=1e-14)


def test_rope_turns():
    for d in (2, 10, 64, 256):
        turns, magnitude = p.rope_turns(d, 5000.0)
        expect = 5000.0 ** (-2.0 * np.arange(d // 2) / d) / (2 * np.pi)
        assert np.allclose(turns, expect, rtol=1e-14) and magnitude == 1.0
        linear, _ = p.rope_turns(d, 5000.0, p.ROPE_SCALE_LINEAR, 8.0)
        assert np.allclose(linear, expect / 8.0, rtol=1e-14)
    # the slowest pair of the changed base turns as the divided one does, the fastest stays
    d = 128
    plain, _ = p.rope_turns(d)
    base, _ = p.rope_turns(d, kind=p.ROPE_SCALE_BASE, factor=4.0)
    assert base[0] == plain[0] and math.isclose(base[-1], plain[-1] / 4.0, rel_tol=1e-12)
    # by parts: fast pairs stay, slow ones are divided, between them everything falls
    parts, magnitude = p.rope_turns(d, kind=p.ROPE_SCALE_PARTS, factor=4.0, context=4096.0)
    assert math.isclose(magnitude, 1 + 0.1 * math.log(4.0), rel_tol=1e-7)
    fast, slow = plain * 4096 >= 34.0, plain * 4096 < 0.85  # a pair away from the borders, which are rounded outwards
    assert np.array_equal(parts[fast], plain[fast]) and fast.any()
    assert np.allclose(parts[slow], plain[slow] / 4.0, rtol=1e-14) and slow.any()
    ratio = parts / plain
    assert np.all(np.diff(ratio) <= 1e-12) and np.all(ratio >= 0.25 - 1e-12)


@pytest.mark.parametrize("change", [
    dict(rotary_dim=0), dict(rotary_dim=3), dict(rotary_dim=1026), dict(base=1.0), dict(base=0.0), dict(base=INF),
    dict(base=NAN), dict(kind=4), dict(kind=1, factor=0.5), dict(kind=1, factor=NAN), dict(kind=2, factor=INF),
    dict(kind=2, rotary_dim=2, factor=2.0), dict(kind=2, rotary_dim=4, base=1e300, factor=1e300),
    dict(kind=3, factor=2.0), dict(kind=3, factor=2.0, context=NAN), dict(kind=3, factor=2.0, context=100.0, slow_turns=0.0),
    dict(kind=3, factor=2.0, context=100.0, fast_turns=1.0, slow_turns=1.0),
    dict(kind=3, factor=2.0, context=100.0, fast_turns=INF), dict(kind=3, factor=2.0, context=100.0, fast_turns=NAN)])
def test_rope_turns_refuses(change):
    with pytest.raises(p.ReactorIssue):
        p.rope_turns(**dict(dict(rotary_dim=64), **change))


def test_rope_turns_refuses_structs(rt):
    s = p.PrometheusRopeScaling(ctypes.sizeof(p.PrometheusRopeScaling), 4, 0, 0, 10.0)
    turns, magnitude = (ctypes.c_double * 2)(), ctypes.c_float()
    call = rt.lib.prometheus_reactor_rope_turns
    assert call(byref(s), turns, byref(magnitude)) == p.PROM_OK
    assert call(None, turns, byref(magnitude)) == call(byref(s), None, byref(magnitude)) == p.PROM_ERROR
    assert call(byref(s), turns, None) == p.PROM_ERROR
    s.reserved0 = 1
    assert call(byref(s), turns, byref(magnitude)) == p.PROM_ERROR
    s.reserved0, s.struct_size = 0, 8
    assert call(byref(s), turns, byref(magnitude)) == p.PROM_ERROR


# ------------------------------------------------------------------ refusals
def _call(rt, name, *args):
    stage, detail = c_uint32(99), c_int(99)
    rc = getattr(rt.lib, name)(rt.handle, *args, byref(stage), byref(detail))
    return rc, stage.value, detail.value


def _refused(result):
    return result == (p.PROM_ERROR, p.STAGE_INIT, p.DETAIL_INVALID_ARGUMENT)


def _no_device(result):
    return result == (p.PROM_ERROR, p.STAGE_INIT, p.DETAIL_HIP_UNAVAILABLE)


def _struct(cls, values, **change):
    if values is None:
        return None
    s = cls()
    s.struct_size = ctypes.sizeof(cls)
    for name, value in dict(values, **change).items():
        setattr(s, name, value)
    return byref(s)


MATRIX = dict(n=48, k=300, group=64, count=1, data=OK)
BAD_MATRICES = [dict(struct_size=8), dict(n=0), dict(n=(1 << 24) + 1), dict(k=0), dict(k=(1 << 20) + 1), dict(group=16),
                dict(group=0), dict(group=256), dict(count=0), dict(count=(1 << 16) + 1), dict(reserved0=1), dict(data=0),
                dict(data=OK + 8)]


def _matrix(**change):
    return _struct(p.PrometheusW4Matrix, MATRIX, **change)


@pytest.mark.parametrize("name", ("pack", "unpack"))
def test_w4_rows_refuse(rt, name):
    call = lambda m, w=OK, stride=300, dtype=p.DTYPE_F32: _call(  # noqa: E731
        rt, f"prometheus_reactor_runtime_w4_{name}_device", m, w, stride, dtype)
    for change in BAD_MATRICES:
        assert _refused(call(_matrix(**change))), change
    assert _refused(call(None))
    for change in (dict(w=0), dict(w=OK + 2), dict(stride=299), dict(stride=1 << 24), dict(dtype=2),
                   dict(w=OK + 1, dtype=p.DTYPE_BF16)):
        assert _refused(call(_matrix(), **change)), change
    for change in ({}, dict(stride=(1 << 24) - 1), dict(w=OK + 2, dtype=p.DTYPE_BF16)):
        assert _no_device(call(_matrix(count=9), **change)), change


GEMM = dict(dtype=p.DTYPE_BF16, rows=5, x_stride=300, out_stride=48, x=OK, out=OK)


def test_gemm_w4_refuses(rt):
    call = lambda m, r: _call(rt, "prometheus_reactor_runtime_gemm_w4_device", m, r)  # noqa: E731
    request = lambda **change: _struct(p.PrometheusW4GemmRequest, GEMM, **change)  # noqa: E731
    assert _refused(call(None, request())) and _refused(call(_matrix(), None))
    for change in BAD_MATRICES:
        assert _refused(call(_matrix(**change), request())), change
    for change in (dict(struct_size=4), dict(dtype=2), dict(rows=0), dict(rows=(1 << 20) + 1), dict(x_stride=299),
                   dict(x_stride=1 << 24), dict(out_stride=47), dict(out_stride=1 << 24), dict(reserved0=1), dict(x=0),
                   dict(x=OK + 1), dict(out=0), dict(out=OK + 1), dict(dtype=p.DTYPE_F32, x=OK + 2)):
        assert _refused(call(_matrix(), request(**change))), change
    assert _no_device(call(_matrix(), request()))
    assert _no_device(call(_matrix(count=3), request(rows=1 << 20, x=OK + 2, out=OK + 6)))


MOE = dict(dtype=p.DTYPE_F32, tokens=3, top_k=2, x_stride=300, out_stride=300, activation=0, renormalise=1, router=OK, x=OK,
           out=OK)


def test_moe_refuses(rt):
    def call(gate={}, up={}, down={}, request={}):
        matrices = []
        for change, n, k in ((gate, 48, 300), (up, 48, 300), (down, 300, 48)):
            matrices.append(None if change is None else _struct(
                p.PrometheusW4Matrix, dict(n=n, k=k, group=64, count=8, data=OK), **change))
        r = None if request is None else _struct(p.PrometheusMoeRequest, MOE, **request)
        return _call(rt, "prometheus_reactor_runtime_moe_w4_device", *matrices, r)

    assert _no_device(call())
    assert _no_device(call(down=dict(group=32), request=dict(out_experts=OK, out_weights=OK, top_k=8)))
    for name in ("gate", "up", "down", "request"):
        assert _refused(call(**{name: None})), name
    for name in ("gate", "up", "down"):
        for change in BAD_MATRICES + [dict(count=9), dict(n=47), dict(k=64)]:
            assert _refused(call(**{name: change})), (name, change)
    assert _refused(call(up=dict(group=32)))
    many = dict(count=p.MOE_MAX_EXPERTS + 1)
    assert _refused(call(gate=many, up=many, down=many))
    for change in (dict(struct_size=4), dict(dtype=2), dict(tokens=0), dict(top_k=0), dict(top_k=9),
                   dict(tokens=p.MOE_MAX_PAIRS // 2 + 1), dict(x_stride=299), dict(x_stride=1 << 24),
                   dict(out_stride=299), dict(out_stride=1 << 24), dict(activation=2), dict(renormalise=2),
                   dict(router=0), dict(router=OK + 2), dict(x=0), dict(x=OK + 2), dict(out=0), dict(out=OK + 2),
                   dict(out_experts=OK + 2), dict(out_weights=OK + 1)):
        assert _refused(call(request=change)), change
    full = dict(count=p.MOE_MAX_EXPERTS)
    assert _no_device(call(gate=full, up=full, down=full, request=dict(tokens=1024, top_k=p.MOE_MAX_TOP_K)))
    assert _refused(call(gate=full, up=full, down=full, request=dict(top_k=p.MOE_MAX_TOP_K + 1)))


ROPE = dict(dtype=p.DTYPE_BF16, rows=4, head_dim=80, rotary_dim=40, layout=0, q_heads=6, k_heads=2, q_stride=480,
            k_stride=160, q_out_stride=480, k_out_stride=160, magnitude=1.0, positions=OK, turns=OK, q=OK, k=OK,
            q_out=2 * OK, k_out=3 * OK)


def test_rope_refuses(rt):
    call = lambda **change: _call(rt, "prometheus_reactor_runtime_rope_device",  # noqa: E731
                                  _struct(p.PrometheusRopeRequest, ROPE, **change))
    assert _refused(_call(rt, "prometheus_reactor_runtime_rope_device", None))
    for change in (dict(struct_size=4), dict(dtype=2), dict(rows=0), dict(rows=(1 << 22) + 1), dict(head_dim=1),
                   dict(head_dim=1026, q_stride=1 << 20, q_out_stride=1 << 20, k_stride=1 << 20, k_out_stride=1 << 20),
                   dict(rotary_dim=0), dict(rotary_dim=39), dict(rotary_dim=82), dict(layout=2), dict(magnitude=INF),
                   dict(magnitude=NAN), dict(reserved0=1), dict(positions=0), dict(positions=OK + 2), dict(turns=0),
                   dict(turns=OK + 4), dict(q=0, q_out=0, k=0, k_out=0), dict(q=0), dict(q_out=0), dict(k=0),
                   dict(k_out=0), dict(q_heads=0), dict(k_heads=(1 << 16) + 1), dict(q_stride=479), dict(k_stride=159),
                   dict(q_out_stride=1 << 24), dict(k_out_stride=159), dict(q=OK + 1), dict(k_out=OK + 1),
                   dict(q_out=OK, q_out_stride=481), dict(dtype=p.DTYPE_F32, k=OK + 2)):
        assert _refused(call(**change)), change
    for change in ({}, dict(q=0, q_out=0, q_heads=0, q_stride=0), dict(k=0, k_out=0), dict(q_out=OK, k_out=OK),
                   dict(q=OK + 2, magnitude=-2.0), dict(rotary_dim=2, layout=1)):
        assert _no_device(call(**change)), change


NORM = dict(dtype=p.DTYPE_F32, rows=4, width=70, h_stride=70, y_stride=71, h_out_stride=72, out_stride=73,
            vector_stride=210, rows_per_vector=2, residual_scale=1.0, eps=1e-6, h=OK, y=2 * OK, post=OK, gate=OK, pre=OK,
            scale=OK, shift=OK, h_out=3 * OK, out=4 * OK)


def test_residual_norm_refuses(rt):
    call = lambda **change: _call(rt, "prometheus_reactor_runtime_residual_norm_device",  # noqa: E731
                                  _struct(p.PrometheusResidualNormRequest, NORM, **change))
    assert _refused(_call(rt, "prometheus_reactor_runtime_residual_norm_device", None))
    wide = p.RESIDUAL_NORM_MAX_WIDTH + 1
    strides = {name: wide for name in ("h_stride", "y_stride", "h_out_stride", "out_stride", "vector_stride")}
    for change in (dict(struct_size=4), dict(dtype=2), dict(rows=0), dict(rows=(1 << 22) + 1), dict(width=0),
                   dict(strides, width=wide), dict(h_stride=69), dict(y_stride=69), dict(h_out_stride=69),
                   dict(out_stride=1 << 24), dict(vector_stride=69), dict(rows_per_vector=0), dict(gate_tanh=2),
                   dict(residual_scale=INF), dict(weight_offset=NAN), dict(eps=-1e-6), dict(eps=NAN), dict(eps=INF), dict(h=0),
                   dict(h=OK + 2), dict(y=OK + 2), dict(post=OK + 2), dict(pre=OK + 1), dict(gate=OK + 2),
                   dict(scale=OK + 1), dict(shift=OK + 2), dict(h_out=0, out=0), dict(h_out=4 * OK), dict(out=OK + 2),
                   dict(h_out=OK), dict(out=2 * OK, out_stride=72)):
        assert _refused(call(**change)), change
    for change in ({}, dict(y=0, y_stride=0), dict(post=0), dict(gate=0, scale=0, shift=0, rows_per_vector=0, vector_stride=0),
                   dict(pre=0), dict(h_out=0), dict(out=0), dict(h_out=OK, h_out_stride=70), dict(out=2 * OK, out_stride=71),
                   dict(dtype=p.DTYPE_BF16, h=OK + 2, gate=OK + 6), dict(strides, width=wide - 1)):
        assert _no_device(call(**change)), change


def test_unknown_handles_are_refused(rt):
    stage, detail = c_uint32(99), c_int(99)
    lib = rt.lib
    calls = [
        lambda: lib.prometheus_reactor_runtime_w4_pack_device(OK, None, OK, 1, 0, byref(stage), byref(detail)),
        lambda: lib.prometheus_reactor_runtime_w4_unpack_device(None, None, OK, 1, 0, byref(stage), byref(detail)),
        lambda: lib.prometheus_reactor_runtime_gemm_w4_device(OK, None, None, None, None),
        lambda: lib.prometheus_reactor_runtime_moe_w4_device(OK, None, None, None, None, byref(stage), byref(detail)),
        lambda: lib.prometheus_reactor_runtime_rope_device(OK, None, byref(stage), byref(detail)),
        lambda: lib.prometheus_reactor_runtime_residual_norm_device(None, None, byref(stage), byref(detail)),
    ]
    for call in calls:
        assert call() == p.PROM_INVALID_HANDLE
    # the wrappers raise what the library refuses
    for call in (lambda: rt.w4_pack_device(p.w4_matrix(0, 1, 1, 32), OK, 1, p.DTYPE_F32),
                 lambda: rt.gemm_w4_device(p.w4_matrix(OK, 1, 1, 32), OK, OK, 0, 1, 1, p.DTYPE_F32),
                 lambda: rt.rope_device(OK, OK, 1, 64, 64, 0, p.DTYPE_F32),
                 lambda: rt.residual_norm_device(0, OK, OK, 1, 1, p.DTYPE_F32)):
        with pytest.raises(p.ReactorIssue):
            call()


def test_struct_layouts_match_the_header(tmp_path):
    header = Path(p.PACKAGE_DIR).parent / "include" / "prometheus_reactor.h"
    classes = (p.PrometheusW4Matrix, p.PrometheusW4GemmRequest, p.PrometheusMoeRequest, p.PrometheusRopeRequest,
               p.PrometheusRopeScaling, p.PrometheusResidualNormRequest)
    names = ("MOE_SILU", "MOE_GELU_TANH", "MOE_MAX_EXPERTS", "MOE_MAX_TOP_K", "MOE_MAX_PAIRS", "ROPE_HALF", "ROPE_PAIRS",
             "ROPE_SCALE_NONE", "ROPE_SCALE_LINEAR", "ROPE_SCALE_BASE", "ROPE_SCALE_PARTS", "RESIDUAL_NORM_MAX_WIDTH")
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void){"]
    expect = []
    for cls in classes:
        lines.append(f'printf("%zu\\n", sizeof({cls.__name__}));')
        expect.append(ctypes.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({cls.__name__}, {field}));')
            expect.append(getattr(cls, field).offset)
    for name in names:
        lines.append(f'printf("%u\\n", (unsigned)PROM_{name});')
        expect.append(getattr(p, name))
    (tmp_path / "l.c").write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(tmp_path / "l"), str(tmp_path / "l.c")], check=True)
    out = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in out] == expect
