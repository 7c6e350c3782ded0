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


def test_barriers_wait_for_lds_reads():
    """A barrier without __syncthreads()'s fences stands between a wave's reads of a stage
    in LDS and other waves' DMA into it: the reads have ended, by an instruction and not by
    the place that the compiler gives to their uses."""
    text = (PKG / "csrc" / "dense.h").read_text()
    body = re.search(r"void block_barrier\(\) \{(.*?)\n\}", text, re.S).group(1)
    assert body.index("s_waitcnt lgkmcnt(0)") < body.index("barrier()")
    for name in ("dense_big.hip", "dense_gemm.hip"):
        text = (PKG / "csrc" / name).read_text()
        text = text[text.index("__global__"):]
        if name == "dense_gemm.hip":
            assert "bare_barrier" not in text and "s_barrier" not in text
        else:  # (each phase waits by itself before its barrier; the second one follows no read)
            assert text.count("bare_barrier()") == 6 and "s_barrier" not in text
            turn = re.search(r"auto turn = .*?\n  \};", text, re.S).group(0)
            assert turn.index("s_waitcnt lgkmcnt(0)") < turn.index("bare_barrier()")
