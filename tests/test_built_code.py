"""The library's device code, disassembled: what a block of inline assembly has to see to by itself, because the compiler
does not look into it."""
from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

from oct_amd import build
from oct_amd import prometheus as p

OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")


def transfers(listing):
    """Each transfer from memory to LDS of an objdump listing, with its kernel and the instructions before it."""
    kernel, before = None, []
    for line in listing.splitlines():
        named = re.match(r"[0-9a-f]+ <(.*)>:", line)
        if named:
            kernel, before = named.group(1), []
            continue
        text = line.split("//")[0].strip()
        if re.match(r"buffer_load\w* .* lds$", text):
            yield kernel, before[-8:], text
        if text:
            before.append(text)


def scalars(operands):
    """The scalar registers that a list of operands names."""
    found = {int(n) for n in re.findall(r"\bs(\d+)\b", operands)}
    for first, last in re.findall(r"\bs\[(\d+):(\d+)\]", operands):
        found |= set(range(int(first), int(last) + 1))
    return found


def too_early(before, transfer):
    """Why the hardware may not yet see what `transfer` reads: m0 written less than one wait state before by a scalar
    instruction, or its descriptor or base less than five before by a vector one."""
    reads, waits = scalars(transfer.split(None, 1)[1]), 0
    for text in reversed(before):
        op, _, operands = text.partition(" ")
        target = operands.split(",")[0]
        if target.strip() == "m0" and waits < 1:
            return text
        if op.startswith("v_") and waits < 5 and scalars(target) & reads:
            return text
        waits += 1 + (int(operands) if op == "s_nop" else 0)
    return None


def test_the_rule():
    load = "buffer_load_dwordx4 v1, s[4:7], s9 offen lds"
    assert too_early(["s_mov_b32 m0, s2"], load) and not too_early(["s_mov_b32 m0, s2", "s_nop 0"], load)
    assert not too_early(["s_mov_b32 m0, s2", "v_add_u32_e32 v1, v2, v3"], load)
    assert too_early(["v_readfirstlane_b32 s9, v0", "s_nop 3"], load) and not too_early(["v_readfirstlane_b32 s9, v0", "s_nop 4"], load)
    assert too_early(["v_readfirstlane_b32 s6, v0"], load) and not too_early(["v_readfirstlane_b32 s8, v0"], load)


@pytest.mark.skipif(not OBJDUMP.exists(), reason="no disassembler")
def test_transfers_to_lds_see_their_registers(tmp_path):
    library = Path(p.PACKAGE_DIR) / build.LIB_PATH.name
    if not library.exists():
        build.build_reactor()
    shutil.copy(library, tmp_path / "library")
    subprocess.run([str(OBJDUMP), "--offloading", "library"], cwd=tmp_path, check=True, capture_output=True)
    found, kernels = 0, set()
    for code in tmp_path.glob(f"library.*{build.ARCH}"):
        listing = subprocess.run([str(OBJDUMP), "-d", "--no-show-raw-insn", str(code)], check=True, capture_output=True, text=True)
        for kernel, before, transfer in transfers(listing.stdout):
            found += 1
            kernels.add(kernel)
            assert too_early(before, transfer) is None, (kernel, before, transfer)
    assert found > 500 and any("w4_tile_kernel" in k for k in kernels)
