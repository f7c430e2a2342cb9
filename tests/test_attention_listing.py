"""The attention of many rows writes its loads to LDS as assembly, which the compiler does not look into.  A vector instruction that writes a scalar register has to be five wait
states before a load from memory that reads it: the compiler sees to that for its own loads only, so the listing is looked over here, along every way that leads to such a load."""
import os
import re
import subprocess

import pytest

from tannic_amd import build

WAIT = 5


def scalars(text):
    """Numbers of the scalar registers in an operand list."""
    found = {int(n) for n in re.findall(r"\bs(\d+)\b", text)}
    for first, last in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        found |= set(range(int(first), int(last) + 1))
    return found


def functions(lines):
    """The instructions (opcode, operands) of every function, labels among them as (None, name)."""
    now = None
    for line in lines:
        label = re.match(r"(_Z\w+|\.LBB\w+):", line)
        text = line.split(";")[0].strip()
        if label and label[1].startswith("_Z"):
            if now:
                yield now
            now = []
        elif label and now is not None:
            now.append((None, label[1]))
        elif now is not None and text and not text.startswith(".") and not text.endswith(":"):
            opcode, _, operands = text.partition(" ")
            now.append((opcode, operands.strip()))
    if now:
        yield now


def too_near(instructions):
    """Loads to LDS, and those of them that read a scalar register which a vector instruction has written less than WAIT states before."""
    labels = {operands: i for i, (opcode, operands) in enumerate(instructions) if opcode is None}
    jumps = {}
    for i, (opcode, operands) in enumerate(instructions):
        if opcode and opcode.startswith(("s_cbranch", "s_branch")):
            jumps.setdefault(labels[operands], []).append(i)
    loads, bad = 0, []
    for i, (opcode, operands) in enumerate(instructions):
        if not opcode or not opcode.startswith("buffer_load") or " lds" not in operands:
            continue
        loads += 1
        needed, ways, seen = scalars(operands), [(i - 1, 0)], {}
        while ways:
            at, states = ways.pop()
            while at >= 0 and states < WAIT and seen.get(at, WAIT) > states:
                seen[at] = states
                before, its = instructions[at]
                if before is None:
                    ways += [(j, states) for j in jumps.get(at, [])]
                    if at and instructions[at - 1][0] in ("s_branch", "s_endpgm", "s_setpc_b64"):
                        break
                else:
                    if before.startswith("v_") and scalars(its.split(",")[0]) & needed:
                        bad.append(f"{before} {its} / {opcode} {operands}")
                        break
                    states += int(its, 0) + 1 if before == "s_nop" else 1
                at -= 1
    return loads, bad


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="no compiler here")
def test_scalar_registers_are_there_when_a_load_reads_them(tmp_path):
    listing = tmp_path / "attention_tile.s"
    subprocess.run([build.HIPCC, *build.FLAGS, "-w", "-S", "--cuda-device-only", os.path.join(build.CSRC, "attention_tile.hip"), "-o", str(listing)], check=True, capture_output=True)
    found = 0
    with open(listing) as f:
        for instructions in functions(f):
            loads, bad = too_near(instructions)
            assert not bad, bad[:3]
            found += loads
    assert found >= 100      # (twelve kernels, some sixteen each)


def test_what_the_look_finds():
    near = [("v_readfirstlane_b32", "s5, v1"), ("s_nop", "2"), ("buffer_load_dwordx4", "v0, s[4:7], 0 offen lds")]
    assert too_near(near) == (1, ["v_readfirstlane_b32 s5, v1 / buffer_load_dwordx4 v0, s[4:7], 0 offen lds"])
    assert too_near([near[0], ("s_nop", "4"), near[2]]) == (1, [])
    assert too_near([("v_readlane_b32", "s7, v1, 3"), ("s_branch", ".LBB0_2"), ("s_mov_b32", "s7, 0"), ("s_nop", "7"), (None, ".LBB0_2"), near[2]])[1]
    assert too_near([("v_cmp_eq_u32_e64", "s[8:9], v1, v2"), near[2]]) == (1, [])
