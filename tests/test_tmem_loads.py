"""Every load from tensor memory and its wait are one asm statement.

The load writes its registers some time before the wait returns; in two
statements the compiler may touch or reuse them in between, which no run shows
reliably.  So this reads the sources (hand-written PTX in csrc)."""
from __future__ import annotations

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "efficient-inference-system_b200" / "csrc"


def asm_statements(text: str) -> list[str]:
    """The text of every asm statement, quotes and nesting respected."""
    out = []
    for m in re.finditer(r"\basm\s*(?:volatile\s*)?\(", text):
        depth, i, quoted = 1, m.end(), False
        while depth:
            c = text[i]
            if quoted:
                i += c == "\\"
                quoted = c != '"'
            elif c == '"':
                quoted = True
            else:
                depth += (c == "(") - (c == ")")
            i += 1
        out.append(text[m.start(): i])
    return out


def test_a_load_waits_in_its_own_statement():
    loads = 0
    for path in sorted(CSRC.glob("*.cu*")):
        for stmt in asm_statements(path.read_text()):
            load, wait = "tcgen05.ld." in stmt, "tcgen05.wait::ld" in stmt
            assert load == wait, f"{path.name}: {stmt[:120]}"
            loads += load
    assert loads >= 2  # the 32- and the 64-column load
