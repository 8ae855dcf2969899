"""Launches that the host code chooses, recorded on the CPU (recorded_launches.h): the grids
of the row kernels for very many rows and of the int8 product for very many columns, and the kernel of
the decoder layer's GeGLU product."""
import subprocess
from pathlib import Path

import pytest

from oct_amd import build
from oct_amd import prometheus as p
from tests.test_quantised_path import PLANNED

HERE = Path(__file__).resolve().parent


def compiled(out, check, *sources):
    # The host half alone: the device code's symbol stays unresolved and unused.
    cmd = [build._hipcc(), "--offload-host-only", f"--offload-arch={build.ARCH}", "-O1", "-std=c++17", "-x", "hip",
           "-no-hip-rt", "-Wl,--unresolved-symbols=ignore-all", f"-I{build.REPO_DIR / 'include'}",
           str(HERE / check), *(str(build.CSRC_DIR / s) for s in sources), "-o", str(out), "-pthread"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    assert proc.returncode == 0, proc.stdout + proc.stderr
    return out


@pytest.fixture(scope="module")
def rows_check(tmp_path_factory):
    return compiled(tmp_path_factory.mktemp("row_launches") / "check", "row_launch_check.cpp", "reduction.hip")


@pytest.fixture(scope="module")
def geglu_check(tmp_path_factory):
    return compiled(tmp_path_factory.mktemp("geglu_launches") / "check", "geglu_launch_check.cpp", "sgemm_f32.hip",
                    "sgemm_rows.hip")


# one, four and sixteen waves per row: 2^26, 2^24 and 2^22 rows are 2^32 threads
@pytest.mark.parametrize("rows,width", [(1, 64), (1000, 3840), ((1 << 24) - 1, 2048), (1 << 24, 1025), (1 << 24, 4096),
                                        ((1 << 22) - 1, 8192), (1 << 22, 4100), (5 << 21, 5000), (1 << 26, 256)])
def test_every_row_is_launched(rows_check, rows, width):
    proc = subprocess.run([str(rows_check), str(rows), str(width)], capture_output=True, text=True, timeout=60)
    assert proc.returncode == 0, proc.stdout + proc.stderr


@pytest.fixture(scope="module")
def int8_check(tmp_path_factory):
    return compiled(tmp_path_factory.mktemp("int8_launches") / "check", "int8_launch_check.cpp")


# few rows: a workgroup of 256 threads takes 16 columns, 2^28 columns are 2^32 threads; many rows: 2^30 of
# them in tiles of 64 would be as many
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 32768, 2048), (16, 2048, 65536), (32, 1 << 27, 31), (1, (1 << 27) + 1, 5),
                                   (1, (1 << 28) - 16, 4), (1, (1 << 28) - 15, 4), (15, (1 << 28) + 5, 15),
                                   (3, 1 << 30, 3), (7, 600000000, 7), (33, 130150523, 33), (1 << 30, 1, 1),
                                   (1 << 30, 3, 3), ((1 << 30) - 64, 2, 1), (4224, 20480, 3840), (2009, 8627, 1177)])
def test_every_column_of_an_int8_product_is_launched(int8_check, m, n, k):
    proc = subprocess.run([str(int8_check), str(m), str(n), str(k)], capture_output=True, text=True, timeout=60)
    assert proc.returncode == 0, proc.stdout + proc.stderr


@pytest.fixture(scope="module")
def kv4_check(tmp_path_factory):
    return compiled(tmp_path_factory.mktemp("kv4_plans") / "check", "kv4_plan_check.cpp")


@pytest.mark.parametrize("name,dtype,dim,heads,group,lengths,new,window,plan", PLANNED, ids=[c[0] for c in PLANNED])
def test_plan_of_an_attention_call(kv4_check, name, dtype, dim, heads, group, lengths, new, window, plan):
    """The plans that the same calls are tested with on the device."""
    args = (int(dtype == p.DTYPE_BF16), dim, heads, group, len(lengths), sum(new), max(new), max(lengths), window)
    proc = subprocess.run([str(kv4_check), *map(str, args)], capture_output=True, text=True, timeout=60)
    splits, prompts, few, sums, pages = map(int, proc.stdout.split())
    assert (splits, prompts, sums, pages) == plan and few == (not prompts or len(lengths) > 1)


# up to 48 rows: the few-rows kernel, or the 64-row tile where it measured faster (a layer of
# 48 tokens, 2048 x 2 * 81920: 555 us and 539; of 16: 448 and 497) and can run
@pytest.mark.parametrize("rows,columns,k,kernel", [
    (1, 16384, 2048, "rows"), (48, 16384, 2048, "rows"), (48, 4096, 1024, "rows"), (16, 81920, 2048, "rows"),
    (48, 81920, 2048, "tiles"), (48, 81890, 2048, "rows"), (48, 81920, 2040, "rows"), (49, 16384, 2048, "tiles"),
    (200, 16384, 2040, "none")])
def test_geglu_kernel_of_a_shape(geglu_check, rows, columns, k, kernel):
    proc = subprocess.run([str(geglu_check), str(rows), str(columns), str(k)], capture_output=True, text=True,
                          timeout=60)
    assert proc.returncode == 0 and proc.stdout.split() == [kernel], proc.stdout + proc.stderr
