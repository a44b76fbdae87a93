"""Wait states of the hand-written copies from memory to LDS.

global_load_lds reads its LDS address from m0, one wait state after a scalar write of m0 at the earliest.
The compiler fills it for its own copies and does not look into inline assembly, so every asm statement
that writes m0 has to hold an s_nop (or another instruction that leaves m0 alone) before the copy."""

import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pytorch-engine_amd", "csrc")
SOURCES = sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.h")))


def _statements(text):
    """The instructions of each asm statement of a source file."""
    for m in re.finditer(r"\basm\s+volatile\s*\(", text):
        lines = []
        at = m.end()
        while True:
            part = re.compile(r'\s*"((?:[^"\\]|\\.)*)"').match(text, at)
            if not part:
                break
            lines.append(part.group(1))
            at = part.end()
        yield [i.strip() for i in re.split(r"\\n|;", "".join(lines).replace("\\t", " ")) if i.strip()]


def _hazards(instructions):
    return [(a, b) for a, b in zip(instructions, instructions[1:])
            if re.match(r"s_\w+ m0\b", a) and "_load_" in b and "lds" in b]


def test_the_check_finds_what_it_looks_for():
    bad = 'asm volatile("s_mov_b32 m0, %3\\n\\tglobal_load_lds_dwordx4 %1, %2\\n\\ts_mov_b32 m0, %0" : : );'
    good = bad.replace("%3\\n\\t", "%3\\n\\ts_nop 0\\n\\t")
    assert [len(_hazards(s)) for s in _statements(bad)] == [1]
    assert [len(_hazards(s)) for s in _statements(good)] == [0]


@pytest.mark.parametrize("path", SOURCES, ids=[os.path.basename(p) for p in SOURCES])
def test_a_copy_to_lds_waits_for_its_address(path):
    found = [h for s in _statements(open(path).read()) for h in _hazards(s)]
    assert not found, found


def test_the_copies_are_seen():
    """The kernels that copy by hand are among the statements looked at."""
    seen = {os.path.basename(p) for p in SOURCES for s in _statements(open(p).read())
            if any("load_lds" in i for i in s)}
    assert {"attend.hip", "gemm.hip"} <= seen
