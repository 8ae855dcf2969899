"""The rest of a decoder's step without a device: what the host code launches, at the ends of its ranges."""
from __future__ import annotations

import subprocess

import pytest

from tests.test_launches import compiled


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
