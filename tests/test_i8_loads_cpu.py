"""The kernels of the 8-bit linear path start while the kernel in front, which may write their operands, still runs.
Loads through the non-coherent path (ld.global.nc: __ldg, or a pointer that is const and __restrict__) are defined
only for memory that nothing writes while the kernel lives, so their sources have none. (No run shows it: the
lines that such a load could find stale are rarely left in an L1.)"""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bert-by-hand_b200", "csrc")


@pytest.mark.parametrize("name", ["linear_i8.cu", "rows_i8.cu"])
def test_no_load_through_the_non_coherent_path(name):
    code = re.sub(r"//[^\n]*|/\*.*?\*/", "", open(os.path.join(CSRC, name)).read(), flags=re.S)
    assert "pdl_wait()" in code
    assert re.findall(r"__ldg|__restrict__|ld\.global[.\w]*\.nc", code) == []
