"""Wait states that gfx9 asks of the program, in the built library's own machine code.

The compiler keeps them in the code that it writes and does not look into inline assembly, so they are looked for in what the library
holds.  Between a scalar write of M0 and a load into LDS, which takes its address from there: 1.  Between a vector instruction's write
of a scalar register and a memory instruction that reads it: 5.  An instruction is one state, s_nop N is N + 1.
"""
import os
import re
import shutil
import subprocess

import pytest

from sgtapose_amd import _lib

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
MEMORY = ("buffer_", "global_", "flat_", "scratch_")


def registers(text):
    """Scalar registers named in an operand list."""
    out = {int(n) for n in re.findall(r"\bs(\d+)\b", text)}
    for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        out.update(range(int(a), int(b) + 1))
    return out


def too_close(lines):
    """-> (loads into LDS seen, list of (line number, text) of instructions that come too early)."""
    loads, bad = 0, []
    before = []                                          # (states it takes, writes M0, scalar registers written by the vector unit), newest last
    for at, line in enumerate(lines):
        text = line.split("//")[0].strip()
        if not text or text.endswith(":"):
            continue
        op, _, rest = text.partition(" ")
        if op.startswith(MEMORY):
            lds = rest.endswith(" lds")
            loads += lds
            reads, states = registers(rest), 0
            for n, m0, written in reversed(before):
                if (lds and m0 and states < 1) or (states < 5 and written & reads):
                    bad.append((at, text))
                    break
                states += n
                if states >= 5:
                    break
        first = rest.split(",")[0]
        if op == "s_branch" or op == "s_endpgm":
            before = []
        else:
            nop = int(rest.strip(), 0) + 1 if op == "s_nop" else 1
            before = before[-5:] + [(nop, op.startswith("s_") and first == "m0", registers(first) if op.startswith("v_") else set())]
    return loads, bad


def test_finds_what_comes_too_early():
    assert too_close(["s_mov_b32 m0, s5", "buffer_load_dwordx4 v1, s[4:7], 0 offen lds"]) == (1, [(1, "buffer_load_dwordx4 v1, s[4:7], 0 offen lds")])
    assert too_close(["s_mov_b32 m0, s5", "s_nop 0", "buffer_load_dwordx4 v1, s[4:7], 0 offen lds"]) == (1, [])
    assert too_close(["v_readfirstlane_b32 s6, v0", "s_nop 3", "buffer_load_dwordx4 v[0:3], v4, s[4:7], 0 offen"])[1]
    assert not too_close(["v_readfirstlane_b32 s6, v0", "s_nop 4", "buffer_load_dwordx4 v[0:3], v4, s[4:7], 0 offen"])[1]
    assert too_close(["v_cmp_eq_u32_e64 s[2:3], v0, v1", "s_mov_b32 s9, s8", "global_load_dword v0, v1, s[2:3]"])[1]


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no disassembler")
def test_the_library_keeps_the_wait_states(tmp_path):
    lib = str(tmp_path / "lib.so")
    shutil.copy(_lib.LIB_PATH, lib)
    subprocess.run([OBJDUMP, "--offloading", lib], check=True, cwd=tmp_path, stdout=subprocess.DEVNULL)
    objects = sorted(p for p in os.listdir(tmp_path) if p.endswith("gfx950"))
    assert objects
    loads, found = 0, []
    for name in objects:
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", name], check=True, cwd=tmp_path, capture_output=True, text=True).stdout
        n, bad = too_close(text.splitlines())
        loads += n
        found += [(name, *b) for b in bad]
    assert loads > 1000                                  # the attention and 8-bit kernels copy their tiles this way
    assert not found, "%d of %d: %s" % (len(found), loads, found[:3])
