"""The rest of a decoder's step without a device, at the ends of its ranges: what the host code launches, the largest weights,
frequencies by parts."""
from __future__ import annotations

import subprocess

import numpy as np
import pytest

from oct_amd import prometheus as p
from oracle import decoder_step as od
from tests.test_launches import compiled


def test_the_largest_weights_that_stay_finite():
    """6 s is finite up to 63 * 2^122 and past fp32's range behind it."""
    most = np.float32(63 * 2.0 ** 122)
    w = np.zeros((2, 32), np.float32)
    w[0, :3], w[1, 0] = (most, -most, most / 3), np.nextafter(most, np.float32(np.inf))
    values = od.w4_values(*od.w4_quantise(w, 32), 32)
    top = float(np.finfo(np.float32).max)
    assert values[0].max() == 63 * 2.0 ** 122 <= top < values[1].max()


@pytest.fixture(scope="module")
def moe_check(tmp_path_factory):
    return compiled(tmp_path_factory.mktemp("moe_launches") / "check", "moe_launch_check.cpp")


def _run(check, *args):
    proc = subprocess.run([str(check), *map(str, args)], capture_output=True, text=True, timeout=120)
    assert proc.returncode == 0, proc.stdout + proc.stderr


@pytest.mark.parametrize("bf16", (0, 1))
@pytest.mark.parametrize("hidden,inner,group", [(128, 64, 32), (2048, 1024, 64), (5, 3, 128), (33000, 24, 128)])
def test_every_mixture_is_launched(moe_check, bf16, hidden, inner, group):
    """No count of tokens, experts and chosen ones leaves a launch without workgroups."""
    _run(moe_check, bf16, -1, hidden, inner, group, 0, 0, 0)


@pytest.mark.parametrize("bf16", (0, 1))
@pytest.mark.parametrize("tokens,experts,top_k", [(1, 8, 2), (64, 64, 8), (100, 16, 2)])
def test_a_failed_launch_of_a_mixture_is_its_last(moe_check, bf16, tokens, experts, top_k):
    """What would read a failed launch's results is not queued, and the call returns its error."""
    _run(moe_check, bf16, 0, 128, 64, 32, tokens, experts, top_k)


def test_a_failed_launch_is_the_last_of_a_mixture_of_many_columns(moe_check):
    """Few tokens whose sums are joined in a launch of their own."""
    _run(moe_check, 1, 0, 70000, 24, 128, 2, 2, 1)


@pytest.mark.parametrize("d,base,context,fast,slow", [
    (128, 10000.0, 100.0, 32.0, 1.0), (128, 10000.0, 4.0, 32.0, 1.0), (64, 10000.0, 2048.0, 32.0, 1.0),
    (8, 1.5, 1e4, 2000.0, 0.01), (8, 10.0, 1e9, 32.0, 1.0), (2, 10000.0, 4096.0, 32.0, 1.0), (1024, 5e5, 8192.0, 4.0, 1.0)])
def test_rope_turns_by_parts_at_their_borders(d, base, context, fast, slow):
    """Contexts so short that no pair turns often, and so long that all do: the borders stay within the pairs' numbers."""
    factor, two_pi = 8.0, 2.0 * np.pi
    got, _ = p.rope_turns(d, base, p.ROPE_SCALE_PARTS, factor, context, fast, slow)
    plain = base ** (-2.0 * np.arange(d // 2) / d) / two_pi
    # pair i turns context * plain_i times; the number i, not whole, that turns t times
    number = lambda t: np.log(context / (two_pi * t)) / np.log(base) * d / 2.0  # noqa: E731
    first, last = max(np.floor(number(fast)), 0.0), min(np.ceil(number(slow)), d - 1.0)
    way = np.clip((np.arange(d // 2) - first) / max(last - first, 0.001), 0.0, 1.0)
    assert np.allclose(got, plain * (1.0 - way + way / factor), rtol=1e-12)
    assert got[0] == pytest.approx(plain[0], rel=1e-12)
