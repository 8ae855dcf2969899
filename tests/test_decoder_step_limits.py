"""The rest of a decoder's step without a device: what the host code launches, at the ends of its ranges."""
from __future__ import annotations

import subprocess

import numpy as np
import pytest

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
