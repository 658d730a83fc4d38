"""Inline assembly names every register that it writes and that no output stands for."""
from __future__ import annotations

import pathlib
import re

CSRC = pathlib.Path(__file__).resolve().parents[1] / "leo_amd" / "csrc"


def statements(text):
    """The bracketed parts of a source's asm statements."""
    for found in re.finditer(r"\basm\b(?:\s+volatile)?\s*\(", text):
        depth, at, quoted = 1, found.end(), False
        while depth:
            c = text[at]
            if c == "\\":
                at += 1
            elif c == '"':
                quoted = not quoted
            elif not quoted:
                depth += {"(": 1, ")": -1}.get(c, 0)
            at += 1
        yield text[found.end():at - 1]


def test_a_written_m0_is_declared():
    seen = 0
    for path in sorted((*CSRC.glob("*.hip"), *CSRC.glob("*.h"))):
        for statement in statements(path.read_text()):
            if re.search(r"\b[sv]_\w+\s+m0\b", statement):
                seen += 1
                assert '"m0"' in statement, (path.name, statement)
    assert seen
