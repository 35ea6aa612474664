"""64-bit shifts by a vector register that is the last one of a kernel's allocation.

Registers are allocated to a wavefront eight at a time. A 64-bit shift whose amount stands in the last of them gave wrong results on the card wherever another
wavefront's registers followed (compaction of a pool's pages: an amount in v15 of 16 registers, wrong now and then where two wavefronts shared a SIMD;
with 24 allocated and the same instructions, never): the amount is read as half of a pair. The compiler knows this of gfx90a and not of gfx950."""
import glob
import os
import re
import shutil
import subprocess

import pytest

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
SHIFT = re.compile(r"v_(?:lshl|lshr|ashr)rev_[bi]64(?:_e\d+)? v\[\d+:\d+\], v(\d+),")
REGISTER = re.compile(r"\bv(?:(\d+)\b|\[(\d+):(\d+)\])")


def doubtful(lines):
    """(64-bit shifts by a vector register, those whose amount is the last of eight registers behind which the kernel uses none)"""
    shifts, bad, name, found, last = 0, [], "", [], -1
    for line in list(lines) + [" <end>:"]:
        if not line.startswith("\t"):
            if re.search(r"<.*>:", line):   # a kernel's or a function's first instruction
                bad += [(name, text) for text, amount in found if amount % 8 == 7 and amount >= last]
                name, found, last = line.strip(), [], -1
            continue
        text = line.split("//")[0].strip()
        for one, lo, hi in REGISTER.findall(text):
            last = max(last, int(one or hi))
        shift = SHIFT.match(text)
        if shift:
            shifts += 1
            found.append((text, int(shift.group(1))))
    return shifts, bad


def test_what_counts_as_doubtful():
    head, by7, by8, more = "0001 <kernel>:", "\tv_lshrrev_b64 v[2:3], v7, v[4:5]", "\tv_lshlrev_b64 v[2:3], v6, v[4:5]", "\tv_mov_b32_e32 v8, v1"
    assert doubtful([head, by7]) == (1, [(head, by7.strip())]) and doubtful([head, by8, "\tv_mov_b32_e32 v7, v1"]) == (1, [])
    assert doubtful([head, by7, more]) == (1, []) and doubtful([head, more, "0002 <other>:", by7])[1]
    assert not doubtful([head, "\tv_lshrrev_b64 v[2:3], 7, v[4:5]", "\tv_lshrrev_b32_e32 v2, v7, v3"])[0]
    assert doubtful([head, "\tv_ashrrev_i64 v[2:3], v15, v[4:5]"])[1]


def test_no_kernel_shifts_by_its_last_register(pkg, tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    pkg.lib()
    shutil.copy(pkg.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    modules = glob.glob(str(tmp_path / "lib.so.*gfx950"))
    assert len(modules) > 1
    dumps = [subprocess.Popen([OBJDUMP, "-d", "--no-show-raw-insn", m], stdout=subprocess.PIPE, text=True) for m in modules]
    total, bad = 0, []
    for d in dumps:
        shifts, some = doubtful(d.stdout)
        assert d.wait() == 0
        total += shifts
        bad += some
    assert total > 0
    assert not bad, f"{len(bad)} of {total}: {bad[:5]}"
