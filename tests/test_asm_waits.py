"""Waits that the compiler does not put into inline assembly.

A memory instruction has to follow a vector instruction's write of a scalar register that it reads (a descriptor from a
lane read or a spilled scalar) by 5 states, and one that loads to LDS a scalar write of m0 by one. The compiler keeps these
distances between instructions of its own, but does not look into inline assembly."""
from __future__ import annotations

import re

import pytest

from modelos_amd.build_lib import CSRC

ASM = re.compile(r"asm\s+volatile\s*\(((?:\s*\"(?:[^\"\\]|\\.)*\")+)\s*:(.*?)\);", re.S)


def statements():
    for path in sorted([*CSRC.glob("*.hip"), *CSRC.glob("*.h")]):
        text = path.read_text()
        for m in ASM.finditer(text):
            code = "".join(re.findall(r"\"((?:[^\"\\]|\\.)*)\"", m.group(1))).encode().decode("unicode_escape")
            lines = [x.strip() for x in re.split(r"[\n;]", code) if x.strip()]
            if lines:
                yield f"{path.name}:{text.count(chr(10), 0, m.start()) + 1}", lines, m.group(2)


def states(lines) -> int:
    return sum(int(x.split()[1]) + 1 if x.startswith("s_nop") else 1 for x in lines)


def scalar_memory(lines, operands) -> bool:
    """Whether a memory instruction takes a scalar operand of the statement's."""
    return any(re.match(r"(buffer|global|flat|scratch)_", x) for x in lines) and re.search(r"\"s\"\s*\(", operands) is not None


def test_the_statements_are_found():
    names = {where.split(":")[0] for where, lines, operands in statements() if any("lds" in x.split() or "_lds_" in x for x in lines)}
    assert {"attn_common.h", "linear_cross_entropy.hip", "score_topk.hip"} <= names


@pytest.mark.parametrize("where,lines,operands", [pytest.param(*s, id=s[0]) for s in statements() if scalar_memory(*s[1:])])
def test_scalar_operands_are_waited_for(where, lines, operands):
    at = next(i for i, x in enumerate(lines) if re.match(r"(buffer|global|flat|scratch)_", x))
    read = set(re.findall(r"%(\d)", lines[at]))
    scalars = {str(i) for i, c in enumerate(re.findall(r"\"(=?&?\{?\w+\}?)\"\s*\(", operands)) if c == "s"}
    if read & scalars:
        assert states(lines[:at]) >= 5, lines


@pytest.mark.parametrize("where,lines,operands", [pytest.param(*s, id=s[0]) for s in statements()
                                                  if any("lds" in x.split() or "_lds_" in x for x in s[1])])
def test_m0_is_waited_for(where, lines, operands):
    at = next(i for i, x in enumerate(lines) if "lds" in x.split() or "_lds_" in x)
    writes = [i for i, x in enumerate(lines[:at]) if re.match(r"s_\w+ m0,", x)]
    begin = writes[-1] + 1 if writes else 0  # else the compiler writes it right before
    assert states(lines[begin:at]) >= 1, lines
