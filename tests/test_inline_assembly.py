"""Inline assembly in the HIP sources names every fixed register that it writes."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "imageni2r_amd", "csrc")
SOURCES = sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.h")))


def statements(text):
    """The asm statements, each from its word to the closing bracket."""
    for m in re.finditer(r"\basm\b(\s+volatile)?\s*\(", text):
        depth, i = 1, m.end()
        while depth:
            if text[i] == '"':  # a string's brackets are no brackets
                i = text.index('"', i + 1)
            depth += {"(": 1, ")": -1}.get(text[i], 0)
            i += 1
        yield text[m.start():i]


def missing(statement):
    """Fixed registers that a statement's instructions write but its list of clobbers does not name."""
    text = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', statement.split(":")[0])).replace("\\n", "\n").replace("\\t", " ")
    written = set()
    for line in re.split(r"[\n;]", text):
        m = re.match(r"\s*[sv]_\w+\s+(m0|vcc|exec|scc|[sv]\d+)\b", line)
        if m and not line.strip().startswith(("s_nop", "s_waitcnt", "v_cmpx")):
            written.add(m.group(1))
    return {r for r in written if f'"{r}"' not in statement.rsplit(":", 1)[-1]}


def test_the_scan():
    assert missing('asm volatile("s_mov_b32 m0, %0\\n\\ts_nop 0" : : "s"(x) : "memory")') == {"m0"}
    assert not missing('asm volatile("s_mov_b32 m0, %0\\n\\ts_nop 0" : : "s"(x) : "memory", "m0")')
    assert not missing('asm volatile("s_waitcnt vmcnt(0)" ::: "memory")')
    assert list(statements('x; asm volatile("a)" : : "s"(f(x))); y')) == ['asm volatile("a)" : : "s"(f(x)))']


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_written_registers_are_named(path):
    with open(path) as f:
        bad = [(s, missing(s)) for s in statements(f.read()) if missing(s)]
    assert not bad, bad
