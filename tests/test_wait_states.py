"""Wait states of the scan's matrix instructions, in the assembly that its sources compile to.

A matrix instruction's result may be used by another kind of instruction, or its registers be
written by one, only after 8 wait states (4 passes and 4).  The compiler puts them in, but has
been seen to leave them out on a path around a branch's body; the kernels then wait themselves
(``settle()`` in csrc/moc_scan.h) or keep branches away.  Every path from every matrix
instruction is followed here, so that such a place cannot come back unseen."""
from __future__ import annotations

import concurrent.futures as cf
import re
import subprocess
from pathlib import Path

import pytest

import build_lib

NEED = 8
_RANGE, _ONE = re.compile(r"\bv\[(\d+):(\d+)\]"), re.compile(r"\bv(\d+)\b")
_STORES = ("ds_write", "buffer_store", "global_store", "scratch_store", "flat_store")


def _registers(text: str) -> frozenset[int]:
    out = {int(m[1]) for m in _ONE.finditer(text)}
    for m in _RANGE.finditer(text):
        out |= set(range(int(m[1]), int(m[2]) + 1))
    return frozenset(out)


def _functions(asm: str):
    """(name, [(opcode, operands)], {label: place}) of each function."""
    name, code, labels = None, [], {}
    for line in asm.splitlines():
        if m := re.match(r"^(_Z\w+|kernel\w*):", line):
            name, code, labels = m[1], [], {}
        elif line.startswith(".Lfunc_end"):
            if name is not None:
                yield name, code, labels
            name = None
        elif name is None:
            continue
        elif m := re.match(r"^(\.LBB\S+):", line):
            labels[m[1]] = len(code)
        elif m := re.match(r"^\s+([a-z]\w+)\s*([^;]*)", line):
            code.append((m[1], m[2]))


def _touched(op: str, operands: str) -> tuple[frozenset[int], frozenset[int]]:
    """Vector registers that an instruction reads or writes, and those that it writes."""
    if op.startswith(_STORES) or op.startswith("v_cmp"):
        return _registers(operands), frozenset()
    return _registers(operands), _registers(operands.split(",")[0])


def hazards(asm: str, need: int = NEED) -> list[str]:
    found = []
    for name, code, labels in _functions(asm):
        def after(i):
            op, operands = code[i]
            if op == "s_endpgm":
                return []
            if op == "s_branch":
                return [labels[operands.strip()]]
            out = [i + 1] if i + 1 < len(code) else []
            return out + ([labels[operands.strip()]] if op.startswith("s_cbranch") else [])

        for i, (op, operands) in enumerate(code):
            if "mfma" not in op:
                continue
            reached: dict[int, int] = {}
            todo = [(j, 0, _registers(operands.split(",")[0])) for j in after(i)]
            while todo:
                j, waited, live = todo.pop()
                if waited >= need or not live or reached.get(j, need) <= waited:
                    continue
                reached[j] = waited
                what, args = code[j]
                step = 1
                if "mfma" in what:  # (the hardware holds one back for the other's result)
                    live = live - _registers(args.split(",")[0])
                elif what.startswith(("v_", "ds_", "buffer_", "global_", "scratch_", "flat_")):
                    touched, written = _touched(what, args)
                    if touched & live:
                        found.append(f"{name}: {op} {operands.strip()} -> {what} {args.strip()} after {waited}")
                        break
                    live = live - written
                elif what == "s_nop":
                    step = int(args.strip(), 0) + 1
                todo += [(k, waited + step, live) for k in after(j)]
    return found


def _compile(source: str) -> str:
    cmd = [build_lib.HIPCC, *build_lib.COMMON_FLAGS, "--cuda-device-only", "-S", str(build_lib.CSRC / source), "-o", "-"]
    return subprocess.run(cmd, check=True, capture_output=True, text=True).stdout


@pytest.mark.skipif(not Path(build_lib.HIPCC).exists(), reason="needs hipcc")
def test_every_path_waits():
    with cf.ThreadPoolExecutor() as ex:
        for source, asm in zip(("moc_scan.hip", "moc_scan_bwd.hip"), ex.map(_compile, ("moc_scan.hip", "moc_scan_bwd.hip"))):
            assert asm.count("v_mfma") > 1000, source
            found = hazards(asm)
            assert not found, (source, len(found), found[:3])


_KERNEL = """
kernel:
\tv_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], 0
\ts_cbranch_scc1 .LBB0_2
\tv_add_f32_e32 v20, v21, v22
\ts_nop 7
.LBB0_2:
{body}
\ts_endpgm
.Lfunc_end0:
"""


@pytest.mark.parametrize("body, bad", [
    ("\tv_mul_f32_e32 v30, v31, v2", True),            # waits only where the branch is not taken
    ("\ts_nop 5\n\tv_mul_f32_e32 v30, v31, v2", True),
    ("\ts_nop 6\n\tv_mul_f32_e32 v30, v31, v2", False),
    ("\tv_mul_f32_e32 v1, v31, v32", True),            # written over
    ("\tbuffer_store_dwordx4 v[0:3], v40, s[0:3], 0 offen", True),
    ("\tv_mul_f32_e32 v30, v31, v4", False),
    ("\tv_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], v[0:3]", False),
])
def test_the_check_sees_a_missing_wait(body, bad):
    assert bool(hazards(_KERNEL.format(body=body))) is bad
