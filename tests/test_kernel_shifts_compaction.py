"""Compaction's kernels, in which a 64-bit shift by a vector register was seen to go wrong, have none: not even one that is right as long as its amount does not
come to stand in the last register."""
import glob
import os
import re
import shutil
import subprocess

import pytest

from test_kernel_shifts import OBJDUMP, SHIFT


def by_kernel(lines):
    """{kernel: its 64-bit shifts by a vector register}"""
    found, name = {}, ""
    for line in lines:
        if not line.startswith("\t"):
            if re.search(r"<.*>:", line):
                name = line.split("<")[1].split(">")[0]
                found[name] = []
        elif SHIFT.match(line.split("//")[0].strip()):
            found[name].append(line.strip())
    return found


def test_compaction_shifts_32_bits(pkg, tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    pkg.lib()
    shutil.copy(pkg.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    kernels = {}
    for module in glob.glob(str(tmp_path / "lib.so.*gfx950")):
        names = subprocess.run([OBJDUMP, "--syms", module], check=True, capture_output=True, text=True).stdout
        if "compact_" in names:
            dump = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", module], check=True, capture_output=True, text=True).stdout
            kernels.update({k: v for k, v in by_kernel(dump.splitlines()).items() if "compact_" in k})
    assert len(kernels) == 5, sorted(kernels)
    assert not any(kernels.values()), {k: v for k, v in kernels.items() if v}
