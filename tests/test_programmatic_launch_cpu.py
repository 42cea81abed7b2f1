"""Kernels that start while the kernel before them still writes what they will read (programmatic dependent launch) may not use read-only loads, whose lines may be
older than the write. What the sources say is all that can be tested: the stale line comes once in thousands of calls."""
import pathlib
import re

import pytest

KERNELS = pathlib.Path(__file__).resolve().parent.parent / "csrc" / "kernels"
FILES = ["flash_attn.cu", "flash_attn_long.cu", "flash_attn_common.cuh", "cross_attn.cu", "rotary.cu"]


def code(name):
    return re.sub(r"//[^\n]*", "", (KERNELS / name).read_text())


@pytest.mark.parametrize("name", FILES)
def test_no_read_only_loads(name):
    text = code(name)
    assert not re.findall(r"__ldg\s*\(|ld\.global(?:\.\w+)*\.nc", text)
    # a read-only parameter that nothing else may point at
    assert not re.findall(r"const\s+[\w:]+(?:\s+[\w:]+)?\s*\*\s*__restrict__\s+\w+", text)


def test_the_patterns_find_what_they_look_for():
    found = "x = __ldg(p); asm(\"ld.global.L1::no_allocate.nc.v4\"); void k(const float* __restrict__ a, const unsigned long long* __restrict__ b, float* __restrict__ c)"
    assert len(re.findall(r"__ldg\s*\(", found)) == 1 and len(re.findall(r"const\s+[\w:]+(?:\s+[\w:]+)?\s*\*\s*__restrict__\s+\w+", found)) >= 1
