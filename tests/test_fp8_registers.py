"""The kernels in 8-bit floating point keep what they hold in registers: none of them moves any to memory and back (the largest dense tile lost a quarter of its
speed to that when a loop around it was not known to run once)."""
from __future__ import annotations

import os
import re
import subprocess

import pytest

from orin_qwen_lossless_amd import build

LLVM = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(build.HIPCC))), "llvm", "bin")
OBJECT = os.path.join(build.OBJ, "kernels_fp8.hip.o")


@pytest.mark.skipif(not (os.path.exists(OBJECT) and os.path.exists(os.path.join(LLVM, "clang-offload-bundler"))), reason="reads the objects of a build")
def test_no_kernel_spills(tmp_path):
    fat, code = str(tmp_path / "fat"), str(tmp_path / "code")
    run = lambda tool, *args: subprocess.run([os.path.join(LLVM, tool), *args], check=True, capture_output=True, text=True).stdout  # noqa: E731
    run("llvm-objcopy", f"--dump-section=.hip_fatbin={fat}", OBJECT, os.devnull)
    run("clang-offload-bundler", "--type=o", "--unbundle", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", f"--input={fat}", f"--output={code}")
    notes = run("llvm-readelf", "--notes", code)
    found = {name: int(count) for name, count in re.findall(r"\.name:\s+(\S+)\n(?:(?!\.name:).)*?\.vgpr_spill_count:\s+(\d+)", notes, re.S)}
    for kernel, instances in (("k_fp8_few", 30), ("k_fp8_many", 32), ("k_add_rmsnorm_fp8", 4), ("k_fp8_down", 1), ("k_fp8_combine", 1), ("k_fp8_rows", 2)):
        mine = {n: c for n, c in found.items() if re.search(rf"\d{kernel}(I|E)", n)}
        assert len(mine) == instances and not any(mine.values()), (kernel, mine)
