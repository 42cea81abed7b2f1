"""Kernels that start while the kernel before them still writes what they will read (programmatic dependent launch) may not use read-only loads, whose lines may be
older than the write. What the sources say is all that can be tested: the stale line comes once in thousands of calls."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "csrc"
FILES = sorted(str(p.relative_to(CSRC)) for folder in ("kernels", "comm") for p in (CSRC / folder).glob("*.cu*"))


def code(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


@pytest.mark.parametrize("name", FILES)
def test_no_read_only_loads(name):
    text = code(name)
    assert not re.findall(r"__ldg\s*\(|ld\.global(?:\.\w+)*\.nc", text)
    # a read-only parameter that nothing else may point at
    assert not re.findall(r"const\s+[\w:]+(?:\s+[\w:]+)?\s*\*\s*__restrict__\s+\w+", text)


def test_all_kernels_are_looked_at():
    assert len(FILES) >= 16 and "kernels/flash_attn_long.cu" in FILES


def test_the_patterns_find_what_they_look_for():
    found = "x = __ldg(p); asm(\"ld.global.L1::no_allocate.nc.v4\"); void k(const float* __restrict__ a, const unsigned long long* __restrict__ b, float* __restrict__ c)"
    assert len(re.findall(r"__ldg\s*\(", found)) == 1 and len(re.findall(r"const\s+[\w:]+(?:\s+[\w:]+)?\s*\*\s*__restrict__\s+\w+", found)) >= 1
