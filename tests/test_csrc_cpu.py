"""The kernels' inline assembly names what it changes (no GPU)."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "toss-next-ctr-prediction_amd", "csrc")


def asm_statements(text):
    """The argument texts of a source's asm statements."""
    for m in re.finditer(r"\basm\s+(?:volatile\s*)?\(", text):
        depth, i, quoted = 1, m.end(), False
        while depth:
            c = text[i]
            if c == "\\":
                i += 1
            elif c == '"':
                quoted = not quoted
            elif not quoted:
                depth += (c == "(") - (c == ")")
            i += 1
        yield text[m.end():i - 1]


def unnamed_m0(text):
    """The asm statements that write m0 and do not say so: the compiler may keep a value of its own there."""
    return [s for s in asm_statements(text)
            if re.search(r"\bs_\w+\s+m0\s*,", s) and not re.search(r':[^:"]*(?:"[^"]*"\s*,\s*)*"m0"[^:]*$', s)]


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.h"))),
                         ids=os.path.basename)
def test_asm_that_writes_m0_names_it(path):
    with open(path) as fh:
        assert unnamed_m0(fh.read()) == []


def test_the_search_itself():
    bad = 'asm volatile("s_mov_b32 m0, %0\\n\\tbuffer_load %1" ::"s"(a), "v"(f(b)) : "memory");'
    assert len(unnamed_m0(bad)) == 1
    assert unnamed_m0(bad.replace('"memory"', '"memory", "m0"')) == [] == unnamed_m0('asm volatile("" ::: "memory");')
