"""Loads from memory to LDS in the built library. They take their LDS address from M0 and, in one form, their
base from a pair of scalar registers. Inside inline assembly the compiler puts no wait states, so the code has to
hold those that the CDNA3 and CDNA4 instruction set manuals ask for: one between a scalar write of M0 and such a
load, five between a vector instruction's write of a scalar register and a load that takes it as its base.

The compiler does not know that the assembly writes M0, which is sound while no code of its own keeps a value there:
nothing but those writes names M0, each has its load behind the wait state, and nothing reads it implicitly."""
import os
import re
import shutil
import subprocess

import pytest

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
REACH = 8  # instructions before a load that can still matter


def _registers(operand):
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    if m:
        return set(range(int(m[1]), int(m[2]) + 1))
    m = re.fullmatch(r"s(\d+)", operand)
    return {int(m[1])} if m else set()


def short_waits(lines):
    """(how many loads to LDS there are, what is wrong) of a listing's instructions."""
    seen, loads, wrong, set_m0 = [], 0, [], None
    for line in lines:
        code = line.split("//")[0].strip()
        if not line.startswith("\t") or not code:
            if line.endswith(">:"):
                seen = []  # another function
            continue
        op, _, rest = code.partition(" ")
        args = [a.strip() for a in rest.split(",")]
        load = "load_lds" in op
        if re.match(r"(s_sendmsg|s_movrel|v_movrel|s_set_gpr_idx|ds_gws|buffer_load\w*.*\blds\b)", code):
            wrong.append(f"{code}: reads M0")
        if set_m0 and not load and op != "s_nop":
            wrong.append(f"{code}: between {set_m0} and the load")
        if re.search(r"\bm0\b", code):
            set_m0 = code
            if not re.match(r"s_mov_b32 m0, s\d+$", code):
                wrong.append(f"{code}: M0 in other code than the loads'")
        elif op != "s_nop":
            set_m0 = None
        if load:
            loads += 1
            base, states = _registers(args[-1].split()[0]), 0
            for o, a in reversed(seen[-REACH:]):
                if o.startswith("s_") and a[0] == "m0" and states < 1:
                    wrong.append(f"{code}: M0 written {states} wait states before")
                if o.startswith("v_") and states < 5 and _registers(a[0]) & base:
                    wrong.append(f"{code}: {o} {a[0]} {states} wait states before")
                states += 1 + (int(a[0], 0) if o == "s_nop" else 0)
        seen.append((op, args))
    return loads, wrong


def test_the_check_itself():
    good = ["\ts_mov_b32 m0, s4", "\ts_nop 0", "\tglobal_load_lds_dwordx4 v[2:3], off"]
    assert short_waits(good) == (1, [])
    assert len(short_waits([good[0], good[2]])[1]) == 1
    base = ["\tv_readfirstlane_b32 s7, v1", "\ts_mov_b32 m0, s4", "\ts_nop 2", "\tglobal_load_lds_dwordx4 v2, s[6:7]"]
    assert len(short_waits(base)[1]) == 1
    base[2] = "\ts_nop 3"
    assert short_waits(base) == (1, [])
    for other in ("\ts_mov_b32 s1, s2", "\tv_readlane_b32 s1, v0, m0", "\ts_movrels_b32 s1, s2", "\tds_gws_barrier v0"):
        assert short_waits([good[0], other, *good[1:]])[1], other


def test_wait_states(tmp_path):
    from nightrun_amd import _lib

    if not os.path.exists(OBJDUMP):
        pytest.skip("no disassembler")
    shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")  # the code objects are written beside it
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    loads, wrong = 0, []
    for f in sorted(tmp_path.glob("lib.so.*gfx950")):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", f.name], cwd=tmp_path, check=True,
                              capture_output=True, text=True).stdout
        n, w = short_waits(text.splitlines())
        loads, wrong = loads + n, wrong + w
    assert loads > 100
    assert not wrong, f"{len(wrong)} of {loads}: {wrong[:5]}"
