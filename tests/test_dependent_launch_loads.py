"""Host check: kernels that may start while the kernel before them still writes (programmatic
dependent launch) read global memory by ordinary loads.  The read-only path is for memory that
nobody writes while the kernel runs: the compiler may move such loads over the wait, and the
wait does not make the earlier kernel's writes visible to them."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "flashmaxsim.jl_b200" / "csrc"


def code(path):
    text = re.sub(r"//[^\n]*|/\*.*?\*/", "", path.read_text(), flags=re.S)
    return text


def included(path, seen):
    if path not in seen:
        seen.add(path)
        for name in re.findall(r'#include "([^"]+)"', path.read_text()):
            if (CSRC / name).exists():
                included(CSRC / name, seen)
    return seen


FILES = sorted(p for p in CSRC.glob("*.cu") if CSRC / "fms_launch.cuh" in included(p, set()))


def test_there_are_such_files():
    assert len(FILES) >= 4


@pytest.mark.parametrize("path", FILES, ids=lambda p: p.name)
def test_ordinary_loads(path):
    for p in sorted(included(path, set())):
        if p.suffix in (".cu", ".cuh") and "dependency_wait" in code(p):
            found = re.findall(r"__ldg|\.nc\b|__restrict__", code(p))
            assert not found, (p.name, found)
