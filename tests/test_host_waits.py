"""The wait states of the built code object, read from its disassembly (llvm-objdump, from the ROCm toolchain). The
compiler puts in those that gfx950 wants between its own instructions, but neither sees nor completes the
instructions of an asm block, so that a missing one there shows only as a rare wrong lane."""
import os
import re
import shutil
import subprocess

import pytest

import sgl_rocm_kv as kv

NEEDED = 2  # wait states from a vector instruction that writes a scalar register to one that reads it


def _registers(operand):
    operand = operand.strip("-| ")
    if operand == "vcc":
        return {"vcc_lo", "vcc_hi"}
    pair = re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    if pair:
        return {f"s{i}" for i in range(int(pair[1]), int(pair[2]) + 1)}
    return {operand} if re.fullmatch(r"s\d+|vcc_lo|vcc_hi", operand) else set()


def _scalar_writes_and_reads(op, args):
    """Scalar registers that a vector instruction writes, and those that it reads."""
    if op.startswith(("v_cmp_", "v_readfirstlane", "v_readlane")):
        out = 1
    elif re.match(r"v_(add|sub|subrev|addc|subb|subbrev)_co_|v_div_scale|v_mad_[ui]64", op):
        out = 2
    else:
        out = 1 if args and not _registers(args[0]) else 0
    writes = set().union(*map(_registers, args[:out])) if out else set()
    return writes, set().union(set(), *map(_registers, args[out:]))


def missing_waits(lines):
    """(function, writer, reader) of every scalar register that is read too soon."""
    function, recent, found = None, [], []  # recent: [wait states since, registers, line]
    for line in lines:
        head = re.match(r"[0-9a-f]+ <(.*)>:", line)
        if head:
            function, recent = head[1], []
            continue
        line = re.match(r"\s+(\S+)\s*(.*?)\s*(//|$)", line)
        if not line:
            continue
        op, args = line[1], [a.strip() for a in re.split(r",(?![^\[]*\])", line[2])] if line[2] else []
        writes = set()
        if op.startswith("v_"):
            writes, reads = _scalar_writes_and_reads(op, args)
            found += [(function, w, f"{op} {line[2]}") for states, own, w in recent if states < NEEDED and own & reads]
        states = int(args[0], 0) + 1 if op == "s_nop" else 1
        recent = [[s + states, own, w] for s, own, w in recent if s + states < NEEDED]
        if op in ("s_branch", "s_endpgm", "s_setpc_b64"):
            recent = []
        if writes:
            recent.append([0, writes, f"{op} {line[2]}"])
    return found


def test_the_rule_itself():
    def found(*body):
        return missing_waits(["0000 <kernel>:"] + ["\t" + x for x in body])

    compare, select = "v_cmp_ne_u32_e32 vcc, 0, v1 // 0", "v_cndmask_b32_e32 v2, v3, v4, vcc // 0"
    assert found(compare, select) and found(compare, "s_nop 0 // 0", select) and found(compare, "v_mov_b32_e32 v9, v8", select)
    assert not found(compare, "s_nop 1 // 0", select) and not found(compare, "s_nop 0", "v_mov_b32_e32 v9, v8", select)
    assert found("v_cmp_gt_u32_e64 s[4:5], v1, v2", "v_cndmask_b32_e64 v2, v3, v4, s[4:5]")
    assert not found("v_cmp_gt_u32_e64 s[4:5], v1, v2", "v_cndmask_b32_e64 v2, v3, v4, s[6:7]")
    assert not found("s_mov_b64 vcc, s[4:5]", select)
    assert not found(compare, "s_branch 12", select)


def test_no_scalar_register_is_read_too_soon():
    objdump = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")
    if not os.path.exists(objdump):
        objdump = shutil.which("llvm-objdump")
    if not objdump:
        pytest.skip("llvm-objdump is not available to read the code object")
    text = subprocess.run([objdump, "-d", "--mcpu=gfx950", kv.CODE_OBJECT_PATH], capture_output=True, text=True, check=True).stdout
    lines = text.splitlines()
    assert sum("v_cndmask" in x for x in lines) > 1000
    found = missing_waits(lines)
    assert not found, (len(found), sorted({f for f, _, _ in found}), found[0])
