"""Every load from tensor memory is waited for in the asm statement that issues it: its registers are not
valid before the wait, and a compiler may move their use up to the end of the statement that defines them."""

from __future__ import annotations

import re

from conftest import ROOT

CSRC = ROOT / "muzo-clip_b200" / "csrc"


def _asm_statements(text: str):
    """The bodies of `asm volatile(...)`, to the closing parenthesis."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"\basm\s+volatile\s*\(", text):
        depth, i, quoted = 1, m.end(), False
        while depth:
            c = text[i]
            if c == '"' and text[i - 1] != "\\":
                quoted = not quoted
            elif not quoted:
                depth += (c == "(") - (c == ")")
            i += 1
        yield text[m.end(): i - 1]


def test_loads_and_their_waits_are_one_statement():
    loads = 0
    for path in sorted(CSRC.glob("*.cu*")):
        for body in _asm_statements(path.read_text()):
            if "tcgen05.ld." in body:
                loads += 1
                assert body.find("tcgen05.wait::ld") > body.find("tcgen05.ld."), (path.name, body[:80])
                assert '"memory"' in body, (path.name, body[:80])
    assert loads >= 4
