"""Checks of the built gfx950 code objects that need no GPU."""
import os
import re
import shutil
import subprocess

import pytest

from gpu_util import vrs

LLVM = "/opt/rocm/llvm/bin"
TARGET = "hipv4-amdgcn-amd-amdhsa--gfx950"


def _instructions(name, tmp_path):
    """Mnemonic and operands of every instruction of a code object, in order."""
    elf = str(tmp_path / "k.elf")
    subprocess.run([f"{LLVM}/clang-offload-bundler", "--type=o", "--unbundle", f"--targets={TARGET}",
                    f"--input={os.path.join(vrs.LIB_DIR, name)}", f"--output={elf}"], check=True)
    text = subprocess.run([f"{LLVM}/llvm-objdump", "-d", "--mcpu=gfx950", elf], check=True, stdout=subprocess.PIPE,
                          text=True).stdout
    lines = (line.split("//")[0].split(None, 1) for line in text.splitlines() if line.startswith("\t"))
    return [(p[0], p[1].strip() if len(p) > 1 else "") for p in lines]


def _scalars(operand):
    """Numbers of the scalar registers of one operand."""
    m = re.fullmatch(r"s(\d+)|s\[(\d+):(\d+)\]", operand.strip())
    if not m:
        return set()
    return {int(m[1])} if m[1] else set(range(int(m[2]), int(m[3]) + 1))


def _early(code):
    """Loads to LDS that follow too soon on what they read: a scalar write of M0 has to be one wait state
    before, a vector instruction's write of a scalar register five.  An instruction is one wait state, s_nop n
    is n + 1."""
    found = []
    for i, (op, args) in enumerate(code):
        if not (op.startswith(("buffer_load", "global_load")) and re.search(r"\blds\b", op + " " + args)):
            continue
        reads = set().union(*(_scalars(a) for a in re.split(r",\s*|\s+", args)))
        states, j = 0, i - 1
        while j >= 0 and states < 5:
            prior, operands = code[j]
            to = operands.split(",")[0]
            if (to == "m0" and states < 1) or (prior.startswith("v_") and _scalars(to) & reads):
                found.append((code[j], code[i]))
                break
            states += int(operands, 0) + 1 if prior == "s_nop" else 1
            j -= 1
    return found


def test_early_loads_are_found():
    load = ("buffer_load_dwordx4", "v7, s[40:43], 0 offen lds")
    m0, lane, add = ("s_mov_b32", "m0, s0"), ("v_readfirstlane_b32", "s41, v9"), ("s_add_i32", "s2, s3, 1")
    assert len(_early([m0, load])) == len(_early([lane, m0, ("s_nop", "0"), load])) == 1
    assert len(_early([lane, ("s_nop", "1"), m0, ("s_nop", "0"), load])) == 1
    assert not _early([lane, ("s_nop", "2"), m0, ("s_nop", "0"), load]) and not _early([m0, add, load])
    assert not _early([m0, ("buffer_load_dwordx4", "v[0:3], v7, s[40:43], 0 offen")])


@pytest.mark.skipif(not shutil.which("llvm-objdump", path=LLVM), reason="no disassembler")
@pytest.mark.parametrize("name", sorted(f for f in os.listdir(vrs.LIB_DIR) if f.endswith(".hsaco")))
def test_loads_to_lds_wait_for_their_scalar_operands(name, tmp_path):
    """The loads stand in inline assembly, where the compiler inserts no wait states."""
    assert not _early(_instructions(name, tmp_path))
