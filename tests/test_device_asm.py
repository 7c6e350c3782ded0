"""Inline assembly in the kernels' sources, read as text."""

from __future__ import annotations

import re

from conftest import PKG


def blocks():
    """(file, instructions) of every asm statement that has any."""
    for path in sorted((PKG / "csrc").iterdir()):
        if path.suffix in (".hip", ".h"):
            for m in re.finditer(r'\basm\s*(?:volatile)?\s*\(\s*((?:"[^"]*"\s*)+)', path.read_text()):
                text = "".join(re.findall(r'"([^"]*)"', m.group(1)))
                lines = [i.strip() for i in re.split(r"\\n|;", text.replace("\\t", " ")) if i.strip()]
                if lines:
                    yield path.name, lines


def test_loads_to_lds_wait_for_m0():
    """A load to LDS takes its address from M0, which it may read one wait state after
    the write at the earliest. The compiler keeps to that in its own code, not within an
    asm statement."""
    seen = 0
    for name, lines in blocks():
        for i, line in enumerate(lines):
            if re.search(r"\blds$", line):
                seen += 1
                before = lines[:i]
                writes = [k for k, b in enumerate(before) if re.match(r"s_\w+ m0\b", b)]
                assert writes and writes[-1] < i - 1, (name, lines)
    assert seen >= 4
