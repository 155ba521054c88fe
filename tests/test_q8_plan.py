"""What the host says of products of 8-bit integers that are not launched (no GPU)."""
import pytest

from hymt2sharp_b200.kernels import build, ops


@pytest.fixture(autouse=True)
def nvcc():
    try:
        build.find_nvcc()
    except build.BuildError as err:
        pytest.skip(str(err))


@pytest.mark.parametrize("tokens", [1, 100])
def test_a_device_without_room_for_a_pair_is_refused(tokens):
    with pytest.raises(ops.KernelError, match="bad arguments"):
        ops.gemm_q8_describe(tokens, 128, 128, False, 1)


@pytest.mark.parametrize("gated", [False, True])
def test_the_smallest_device_has_one_pair(gated):
    assert ops.gemm_q8_describe(100, 128, 1280, gated, 2)["ctas"] >= 2
    assert ops.gemm_q8_describe(5000, 4096, 1280, gated, 3)["ctas"] == 2
