"""Inline asm says which registers it writes: the compiler keeps values in the others
(CPU, from the sources)."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "strict_amd" / "csrc"
SOURCES = sorted(p for p in CSRC.iterdir() if p.suffix in (".hip", ".h"))


def statements(text):
    """The asm statements of a source, each from its keyword to the closing parenthesis."""
    for m in re.finditer(r"\basm\b(?:\s+volatile)?\s*\(", text):
        depth, at, quoted = 1, m.end(), False
        while depth and at < len(text):
            c = text[at]
            if quoted and c == "\\":
                at += 1
            elif c == '"':
                quoted = not quoted
            elif not quoted:
                depth += (c == "(") - (c == ")")
            at += 1
        yield text[m.start():at]


@pytest.mark.parametrize("source", SOURCES, ids=lambda p: p.name)
def test_writes_of_m0_and_scc_are_named(source):
    for s in statements(source.read_text()):
        template, _, rest = s.partition("::") if "::" in s else s.partition(":")
        if re.search(r"s_mov_b32 m0\b", template):
            assert '"m0"' in rest or '{m0}' in rest, s
        if re.search(r"\bs_cmp_", template):
            assert '"scc"' in rest, s


def test_a_statement_that_names_nothing_is_found():
    text = 'f(); asm volatile("s_mov_b32 m0, %1\\n\\t" "x (%0)" ::"v"(a(b)), "s"(c) : "memory"); g();'
    assert len(list(statements(text))) == 1 and list(statements(text))[0].endswith('"memory")')
