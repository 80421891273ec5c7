"""What the compiler does not check in the built kernels.

A scalar register that a vector instruction writes (``v_readfirstlane`` and its like) may be read by a memory instruction five wait states
later at the earliest; M0, which holds the LDS address of a load straight into LDS, is read one wait state after a scalar instruction wrote it.
The compiler sees to both for its own instructions, not in front of inline assembly, and loads straight into LDS are inline assembly here: a
descriptor, an offset or an LDS address that is read too early sends such a load somewhere else, now and then.
"""
import os
import re
import shutil
import subprocess

import pytest

from brainstorm_amd import _lib

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
WAIT_STATES = 5


def scalars(operand):
    """The scalar registers of an operand."""
    several, one = re.fullmatch(r"s\[(\d+):(\d+)\]", operand), re.fullmatch(r"s(\d+)", operand)
    if several:
        return set(range(int(several[1]), int(several[2]) + 1))
    return {int(one[1])} if one else {operand} & {"vcc", "m0"}


def instructions(function):
    """(opcode, operands, address of a branch's target) of a function in disassembly, by address, and the function's name."""
    head = re.match(r"([0-9a-f]{16}) <(.*)>:", function)
    found = {}
    for line in function.split("\n")[1:] if head else ():
        parts = re.match(r"\t(\S+)(.*?)\s*// ([0-9A-F]+):", line)
        if parts:
            to = re.search(r"<[^>]*?(?:\+0x([0-9a-f]+))?>\s*$", line) if "branch" in parts[1] else None
            operands = [o for o in re.split(r"[,\s]+", parts[2].strip()) if o]
            found[int(parts[3], 16)] = (parts[1], operands, int(head[1], 16) + int(to[1] or "0", 16) if to else None)
    return found, head[2] if head else ""


def read_too_early(code):
    """The loads into LDS of ``instructions`` and, of them, those that read a scalar too early, on any way to them."""
    at = list(code)
    number = {address: i for i, address in enumerate(at)}
    before = [[] for _ in range(len(at) + 1)]
    for i, address in enumerate(at):
        opcode, _, to = code[address]
        if opcode not in ("s_branch", "s_endpgm", "s_setpc_b64"):
            before[i + 1].append(i)
        if to in number:
            before[number[to]].append(i)
    loads, early = 0, []
    for i, address in enumerate(at):
        opcode, operands, _ = code[address]
        if not opcode.startswith("buffer_load") or "lds" not in operands:
            continue
        loads += 1
        read = set().union({"m0"}, *map(scalars, operands))
        ways, seen = [(p, 0) for p in before[i]], set()
        while ways:
            j, states = ways.pop()
            if states >= WAIT_STATES or (j, states) in seen:
                continue
            seen.add((j, states))
            writer, given, _ = code[at[j]]
            if writer.startswith("s_") and states < 1 and given[:1] == ["m0"]:
                early.append(f"{address:#x} {opcode} {operands} right after {writer} {given}")
            if writer.startswith("v_") and any(scalars(o) & read for o in given[:2 if "_co_" in writer or "div_scale" in writer else 1]):
                early.append(f"{address:#x} {opcode} {operands} {states} wait states after {writer} {given}")
            ways += [(p, states + (int(given[0], 0) + 1 if writer == "s_nop" else 1)) for p in before[j]]
    return loads, early


def test_the_check_finds_what_it_looks_for():
    text = """0000000000001000 <kernel>:
\tv_readfirstlane_b32 s10, v2                                // 000000001000: 7E140502
\ts_mov_b32 m0, s4                                           // 000000001004: BEFC0004
\ts_nop 2                                                    // 000000001008: BF800002
\tbuffer_load_dword v1, s[8:11], 0 offen lds                 // 00000000100C: E0511000
\tv_readlane_b32 s7, v3, 0                                   // 000000001014: D2890007
\ts_cbranch_scc1 65530                                       // 00000000101C: BF85FFFA <kernel+0x8>
\tbuffer_load_dwordx4 v1, s[12:15], s7 offen lds             // 000000001020: E05D1000
\ts_nop 4                                                    // 000000001028: BF800004
\tbuffer_load_dwordx4 v1, s[12:15], s7 offen lds             // 00000000102C: E05D1000
\ts_endpgm                                                   // 000000001034: BF810000
"""
    code, name = instructions(text)
    loads, early = read_too_early(code)
    assert (name, loads, [line.split()[0] for line in early]) == ("kernel", 3, ["0x100c", "0x1020"])
    at_once = text.replace("s_mov_b32 m0, s4 ", "s_nop 4 ").replace("s_nop 2 ", "s_mov_b32 m0, s4 ")
    assert "0x100c buffer_load_dword ['v1', 's[8:11]', '0', 'offen', 'lds'] right after s_mov_b32 ['m0', 's4']" in read_too_early(instructions(at_once)[0])[1]
    later = text.replace("s_nop 2 ", "s_nop 3 ")
    assert [line.split()[0] for line in read_too_early(instructions(later)[0])[1]] == ["0x1020"]
    back = later.replace("s7, v3", "s9, v3")  # (what the branch back leads to)
    assert [line.split()[0] for line in read_too_early(instructions(back)[0])[1]] == []
    assert [line.split()[0] for line in read_too_early(instructions(back.replace("s_nop 3 ", "s_nop 1 "))[0])[1]] == ["0x100c", "0x100c"]


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no disassembler")
def test_loads_into_lds_read_scalars_after_their_wait_states(tmp_path):
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("the library is not built")
    library = shutil.copy(_lib.LIB_PATH, tmp_path / "library.so")
    subprocess.run([OBJDUMP, "--offloading", str(library)], check=True, capture_output=True, cwd=tmp_path)
    loads, early = 0, []
    for image in sorted(tmp_path.glob("*amdgcn*")):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(image)], check=True, capture_output=True, text=True).stdout
        for function in re.split(r"\n(?=[0-9a-f]{16} <)", text):
            if " lds" not in function:
                continue
            code, name = instructions(function)
            found, bad = read_too_early(code)
            loads += found
            early += [f"{name} {line}" for line in bad]
    assert loads > 1000, "the kernels that load into LDS were not found"
    assert not early, "\n".join(early[:20])
