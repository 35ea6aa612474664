"""What the built kernels' instructions have to keep, and no pass of the compiler sees to where they stand in inline assembly."""
import glob
import os
import re
import shutil
import subprocess

import pytest

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def scalars(text):
    """Numbers of the scalar registers that an operand names"""
    found = set()
    for one, lo, hi in re.findall(r"\bs(?:(\d+)\b|\[(\d+):(\d+)\])", text):
        found |= {int(one)} if one else set(range(int(lo), int(hi) + 1))
    return found


def too_close(lines):
    """(loads to LDS, those that stand too close behind what they read). M0 holds the place in LDS that a load goes to: a scalar write
    of it takes a wait state to reach the load. A scalar register that a vector instruction has written takes five to reach a memory
    instruction. An instruction is one wait state, s_nop n is n + 1."""
    loads, close, back = 0, [], []   # back: (instruction, wait states that it stands for), the newest first
    for line in lines:
        if not line.startswith("\t"):
            back = []   # a kernel's or a function's first instruction
            continue
        text = line.split("//")[0].strip()
        if "_load_lds" in text or re.search(r"\blds$", text):
            loads += 1
            reads, states = scalars(text.split(" ", 1)[1]), 0
            for before, each in back:
                if states < 1 and re.match(r"s_\w+ m0\b", before):
                    close.append((before, text))
                written = before.split(" ", 1)[1].split(",")[0] if before.startswith("v_") and " " in before else ""
                if reads & scalars(written):
                    close.append((before, text))
                states += each
                if states >= 5:
                    break
        nop = re.match(r"s_nop (\d+)", text)
        back = [(text, int(nop.group(1)) + 1 if nop else 1)] + back[:5]
    return loads, close


def test_what_counts_as_too_close():
    load, off = "\tglobal_load_lds_dwordx4 v4, s[6:7]", "\tglobal_load_lds_dwordx4 v[4:5], off"
    m0, lane, add = "\ts_mov_b32 m0, s3", "\tv_readlane_b32 s7, v9, 1", "\ts_add_u32 s8, s8, s9"
    assert too_close([m0, load]) == (1, [(m0.strip(), load.strip())]) and too_close([m0, off])[1]
    assert not too_close([m0, "\ts_nop 0", load])[1] and not too_close([m0, add, off])[1]
    assert too_close([lane, m0, "\ts_nop 2", load])[1] and not too_close([lane, m0, "\ts_nop 3", load])[1]
    assert not too_close([lane, m0, "\ts_nop 0", off])[1] and too_close([lane, add, add, add, add, load])[1]
    assert not too_close([lane, add, add, add, add, add, load])[1] and not too_close(["0001 <kernel>:", load])[1]


def test_loads_to_lds_wait_for_what_they_read(pkg, tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    pkg.lib()
    shutil.copy(pkg.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    modules = glob.glob(str(tmp_path / "lib.so.*gfx950"))
    assert len(modules) > 1
    dumps = [subprocess.Popen([OBJDUMP, "-d", "--no-show-raw-insn", m], stdout=subprocess.PIPE, text=True) for m in modules]
    total = 0
    for d in dumps:
        loads, close = too_close(d.stdout)
        assert d.wait() == 0
        assert not close, f"{len(close)} of {loads}: {close[:3]}"
        total += loads
    assert total > 0
