"""Properties of the CUDA sources that a compiler may rely on."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "vibeblade_b200" / "csrc"
FILES = sorted(p.name for p in CSRC.iterdir() if p.suffix in (".cu", ".cuh"))


def statements(text):
    """The asm statements of a source, comments taken out."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"\basm\s+volatile\s*\(|\basm\s*\(", text):
        depth, i = 1, m.end()
        quoted = False
        while depth:
            c = text[i]
            if c == '"' and text[i - 1] != "\\":
                quoted = not quoted
            elif not quoted:
                depth += (c == "(") - (c == ")")
            i += 1
        yield text[m.start():i]


@pytest.mark.parametrize("name", FILES)
def test_asynchronous_copies_are_ordered_for_the_compiler(name):
    """A copy into shared memory, its commit and the wait for it say that they touch memory: else the
    compiler may move reads of the copied bytes above the wait."""
    loose = [s for s in statements((CSRC / name).read_text()) if "cp.async" in s and '"memory"' not in s]
    assert not loose, loose


@pytest.mark.parametrize("name", FILES)
def test_waits_are_bounded_in_time(name):
    """A loop over mbarrier tries looks at the clock (how long a try is suspended is the hardware's choice,
    so a number of tries bounds nothing), or at a flag that one which does raises."""
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    loops = [text[m.start():m.start() + 200] for m in re.finditer(r"while \(!mbar_try_wait\w*\(", text)]
    timed = [t for t in loops if "clock" in t]
    assert all(t in timed or (timed and "abort_flag" in t) for t in loops), loops
