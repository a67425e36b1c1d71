"""Kernels that start while earlier ones run read by plain loads only; no GPU needed.

A read-only load (``__ldg``, ``ld.global.nc``, a ``const __restrict__`` pointer) may be
moved before the kernel's wait, or find in L1 what stood there before an earlier kernel
wrote it.
"""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ozaki_triton_b200", "csrc")
WAITS = re.compile(r"griddepcontrol\.wait|start_after_earlier_kernels\(\)|ProgrammaticStreamSerialization"
                   r'|#include "oz_(tile|operands|stream|linear)\.cuh"')
READ_ONLY = re.compile(r"__ldg\s*\(|\.nc\b|\bconst\s+\w+\s*\*\s*__restrict__")


def code_of(name):
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


UNITS = sorted(n for n in os.listdir(CSRC) if n.endswith((".cu", ".cuh")) and WAITS.search(code_of(n)))


def test_the_units_are_found():
    assert {"oz_w4.cu", "oz_experts.cu", "oz_linear.cu", "oz_linear_split.cu", "oz_route.cu", "oz_clip.cu", "oz_newton.cu",
            "oz_tile.cuh", "oz_operands.cuh"} <= set(UNITS)


@pytest.mark.parametrize("name", UNITS)
def test_no_read_only_loads(name):
    found = [line.strip() for line in code_of(name).splitlines() if READ_ONLY.search(line)]
    assert not found, found
