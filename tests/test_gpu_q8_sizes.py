"""Products of 8-bit integers at the ends of the sizes that are taken."""
import pytest
import torch

from test_gpu_kernels import DEV, _ops

pytestmark = pytest.mark.gpu

F32, BF = torch.float32, torch.bfloat16


@pytest.mark.parametrize("N", [5, 8])
def test_more_tokens_than_65535_tiles(N):
    """Rows that TMA writes and rows that it does not: all of them, and the row behind the last."""
    ops = _ops()
    T, K = 256 * 65536 + 300, 16
    g = torch.Generator(device=DEV).manual_seed(N)
    a, w = (torch.randint(-128, 128, (rows, K), generator=g, device=DEV, dtype=torch.int8) for rows in (T, N))
    sa, sw = torch.rand(T, generator=g, device=DEV) + 0.5, torch.rand(N, generator=g, device=DEV) + 0.5
    status = torch.zeros(4, dtype=torch.int32, device=DEV)
    sums = a.float() @ w.float().T            # (whole numbers below 2^18, and their parts: exact)
    assert not torch.backends.cuda.matmul.allow_tf32
    for epilogue, dtype in ((ops.EPILOGUE_STORE, BF), (ops.EPILOGUE_ACCUMULATE, F32)):
        out = torch.ones(T + 1, N, dtype=dtype, device=DEV)
        ops.gemm_q8_tc(out[:T], a, sa, w, sw, epilogue, status)
        want = sums.double() * sa.double()[:, None] * sw.double()
        size = want.abs()
        if epilogue == ops.EPILOGUE_ACCUMULATE:
            want += 1.0
            size += 1.0
        # two products and an addition in float32, one rounding to the output's type
        assert ((out[:T].double() - want).abs() <= (3 * 2.0 ** -24 + torch.finfo(dtype).eps / 2) * 1.01 * size).all()
        assert (out[T] == 1.0).all()
    assert status.tolist() == [0, 0, 0, 0]
