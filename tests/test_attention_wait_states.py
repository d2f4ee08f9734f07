"""The wait states that the direct LDS loads of attention need and that the compiler does not add inside an assembly
statement, read from the assembly that is built here.

On this target a scalar write of m0 needs one wait state before a load to LDS takes its address from it, and a scalar register
written by a vector instruction needs five before a buffer load reads it.  Any instruction is one, ``s_nop n`` is n + 1.
"""
import re
import subprocess

import pytest

from transformer_amd import build


def _scalars(text):
    found = {int(n) for n in re.findall(r"\bs(\d+)\b", text)}
    for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        found |= set(range(int(a), int(b) + 1))
    return found | ({106, 107} if re.search(r"\bvcc\b", text) else set())


def _wait_states(instruction):
    name, *rest = instruction.split(None, 1)
    return int(rest[0], 0) + 1 if name == "s_nop" else 1


def _written_by_vector(instruction):
    """Scalar registers that a vector instruction writes (the first operands that are scalar)."""
    if not instruction.startswith("v_") or " " not in instruction.replace("\t", " "):
        return set()
    operands = re.split(r",\s*", instruction.split(None, 1)[1])
    if instruction.startswith(("v_readfirstlane", "v_readlane", "v_cmp")):
        return _scalars(operands[0])
    return _scalars(operands[1]) if re.match(r"v_(add|sub|subrev|addc|subb|mad_u64|mad_i64|div_scale)", instruction) and len(operands) > 4 else set()


def hazards(assembly):
    """(loads to LDS, what each lacks)."""
    lines = [re.split(r";|//", x)[0].strip() for x in assembly.splitlines()]
    lines = [x for x in lines if x and not x.startswith(".") and not x.endswith(":")]
    loads, lacks = 0, []
    for i, load in enumerate(lines):
        if not re.match(r"buffer_load\w*\s.*\blds$", load):
            continue
        loads += 1
        reads, waited = _scalars(load), 0
        for before in reversed(lines[max(i - 6, 0):i]):
            if waited < 1 and re.match(r"s_\w+\s+m0\b", before):
                lacks.append((before, load))
            if waited < 5 and _written_by_vector(before) & reads:
                lacks.append((before, load))
            waited += _wait_states(before)
    return loads, lacks


LOAD = "\tbuffer_load_dwordx4 v3, s[16:19], 0 offen lds\n"


@pytest.mark.parametrize("before,lacking", [
    ("s_mov_b32 m0, s4\n", True),
    ("s_mov_b32 m0, s4\n;;#ASMEND\n", True),
    ("s_mov_b32 m0, s4\ns_nop 0\n", False),
    ("s_mov_b32 m0, s4\nv_add_u32_e32 v1, v2, v3\n", False),
    ("v_readfirstlane_b32 s17, v1\ns_mov_b32 m0, s4\ns_nop 0\n", True),
    ("v_readfirstlane_b32 s17, v1\ns_nop 3\n", True),
    ("v_readfirstlane_b32 s17, v1\ns_nop 4\n", False),
    ("v_readfirstlane_b32 s20, v1\ns_nop 0\n", False),
])
def test_the_rule(before, lacking):
    assert hazards(before + LOAD)[0] == 1 and bool(hazards(before + LOAD)[1]) == lacking


def test_direct_lds_loads_wait(tmp_path):
    out = tmp_path / "attn.s"
    flags = [f for f in build.HIPCC_FLAGS if f != "-shared"]
    subprocess.run([build.hipcc(), *flags, "--cuda-device-only", "-S", f"{build.HERE}/csrc/attn.hip", "-o", str(out)], check=True)
    loads, lacks = hazards(out.read_text())
    assert loads > 100 and not lacks, lacks[:4]
