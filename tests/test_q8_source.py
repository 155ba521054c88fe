"""What the sources of the 8-bit kernels must not hold (no GPU)."""
import os
import re

import pytest

from hymt2sharp_b200.kernels import build


def _code(name):
    """A source of the library without its comments."""
    with open(os.path.join(build.CSRC, name)) as fh:
        text = fh.read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


@pytest.mark.parametrize("name", ["gemm_q8.cu", "q8_rows.cu"])
def test_nothing_that_a_kernel_in_front_writes_is_read_as_read_only_data(name):
    """These kernels start while the kernel in front of them still runs, and all that they read but settled weights (which come by TMA) may be written by it.
    A read-only load is defined only for what nobody writes while the kernel lives, and may be moved in front of the wait."""
    code = _code(name)
    assert "pdl_wait" in code
    assert not re.search(r"__ldg|ld\.global\.nc|__restrict__|ld\.global(\.\w+)*\.nc", code)
