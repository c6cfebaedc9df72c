"""What the kernels' sources have to say to the compiler, read from their text."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "shelfgaussian-cudagaussianvoxelizer_amd", "csrc")
FILES = sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.h")))


def _statements(text):
    """The inline assembly statements of a source: from `asm` to the semicolon behind its closing bracket."""
    for m in re.finditer(r"\basm\b(?:\s+volatile)?\s*\(", text):
        depth, quoted, i = 1, False, m.end()
        while depth:
            c = text[i]
            if c == '"' and text[i - 1] != "\\":
                quoted = not quoted
            elif not quoted:
                depth += (c == "(") - (c == ")")
            i += 1
        yield text[m.start():i]


@pytest.mark.parametrize("path", FILES, ids=[os.path.basename(p) for p in FILES])
def test_assembly_that_writes_m0_says_so(path):
    """The compiler may keep a value of its own in m0 across a statement that does not list it as written."""
    for s in _statements(open(path).read()):
        if re.search(r"\bm0\s*,", s):
            assert re.search(r':[^:]*"m0"[^:]*\)$', s), s


def test_statements_are_found():
    text = 'x; asm volatile("s_mov_b32 m0, %0\\n\\t(" ::"s"(f(1)) : "memory"); y; asm("s_nop 0");'
    assert [s[-3:] for s in _statements(text)] == ['y")', '0")']
