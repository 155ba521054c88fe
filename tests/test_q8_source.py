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


def test_a_warp_answers_for_all_its_lanes_before_it_reads_tensor_memory():
    """A wait that gives up does so lane by lane, and a load of tensor memory takes the whole warp: between the two stands a vote."""
    waits = re.findall(r"mbar_wait\((?:done_bar|acc_full0).*?;\s*(.*?);", _code("gemm_q8.cu"), flags=re.S)
    assert len(waits) == 2 and all("__all_sync(0xffffffffu" in behind for behind in waits)


def test_every_wait_has_a_limit_that_a_launch_can_give():
    waits = [text.split(";")[0] for text in _code("gemm_q8.cu").split("mbar_wait(")[1:]]
    assert len(waits) == 7 and all("wait_limit<FAULT>(p))" in w for w in waits)
