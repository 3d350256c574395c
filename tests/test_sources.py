"""CPU checks of the kernels' sources themselves: what no output shows until the compiler's choices change."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sandyrt_amd", "csrc")
SOURCES = sorted(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.hip")))


def asm_statements(text):
    """The arguments of every asm statement, brackets matched (those inside their strings come in pairs)."""
    for m in re.finditer(r"\basm\s*(?:volatile)?\s*\(", text):
        depth, end = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[end], 0)
            end += 1
        yield text[m.end():end - 1]


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_assembly_that_writes_m0_says_so(path):
    """Else the compiler may keep a value of its own there across the statement."""
    for body in asm_statements(open(path).read()):
        if re.search(r"\bs_\w+\s+m0\b", body):
            assert '"m0"' in body, body
