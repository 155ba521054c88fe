"""Products of 8-bit integers in which one wait runs out: a k block is announced and never copied.  The kernel must say so, write no number (of few tokens
NaN, of many nothing), free its tensor memory and return; the next products are right."""
import pytest
import torch

from test_gpu_kernels import DEV, _ops

pytestmark = pytest.mark.gpu

F32, BF = torch.float32, torch.bfloat16


def _operands(T, rows_w, K, seed):
    ops = _ops()
    g = torch.Generator(device=DEV).manual_seed(seed)
    a, w = ops.q8_rows(T, K, DEV), ops.q8_rows(rows_w, K, DEV)
    for m in (a, w):
        m.copy_(torch.randint(-128, 128, m.shape, generator=g, device=DEV, dtype=torch.int8))
    return a, torch.rand(T, generator=g, device=DEV) + 0.5, w, torch.rand(rows_w, generator=g, device=DEV) + 0.5


# one CTA; K cut over a cluster, then by more blocks than the ring has stages; two pairs of CTAs (gated: four), and three with a ring that comes round
SHAPES = [(8, 128, 256, dict(few=1, splits=1)), (8, 128, 2048, dict(few=1, splits=8)), (16, 128, 16384, dict(few=1, splits=8)),
          (300, 64, 384, dict(few=0, splits=1)), (520, 32, 2048, dict(few=0, splits=1))]


@pytest.mark.parametrize("epilogue, dtype", [(1, F32), (2, BF)])
@pytest.mark.parametrize("T, N, K, plan", SHAPES)
def test_a_wait_that_runs_out_is_reported_and_no_number_is_written(T, N, K, plan, epilogue, dtype):
    ops = _ops()
    gated = epilogue == ops.EPILOGUE_SWIGLU
    how = ops.gemm_q8_describe(T, N, K, gated)
    assert {k: how[k] for k in plan} == plan and how["ctas"] <= 8 and (how["stages"] < how["k_blocks"]) == (K > 2048 or T == 520)
    rows_w = 2 * N if gated else N
    a, sa, w, sw = _operands(T, rows_w, K, T + K)
    status = torch.zeros(4, dtype=torch.int32, device=DEV)
    base = torch.randn(T, N, device=DEV).to(dtype)
    for block in sorted({1, K // 128 - 1}):
        out = base.clone()
        ops.gemm_q8_debug(out, a, sa, w, sw, epilogue, status, 4096, block)
        torch.cuda.synchronize()                         # the kernel came back
        assert status.tolist()[0] in (151, 152, 153) and status.tolist()[1:] == [0, 0, 0]
        assert torch.isnan(out).all() if how["few"] else torch.equal(out, base)
        status.zero_()
    for _ in range(20):                                  # (tensor memory that was not freed would be missing by now)
        out = base.clone()
        ops.gemm_q8_tc(out, a, sa, w, sw, epilogue, status)
    assert status.tolist() == [0, 0, 0, 0]
    if gated:
        return
    want = (a.double() @ w.double().T) * sa.double()[:, None] * sw.double() + base.double()
    # the sum to float32, two products, an addition: four half steps of float32
    assert ((out.double() - want).abs() <= 4 * 2.0 ** -24 * 1.01 * (want.abs() + base.double().abs())).all()


def test_launches_that_take_no_fault():
    ops = _ops()
    status = torch.zeros(4, dtype=torch.int32, device=DEV)
    a, sa, w, sw = _operands(8, 4096, 256, 1)
    out = torch.zeros(8, 4096, device=DEV)
    for out_, epilogue, what in ((out.bfloat16(), ops.EPILOGUE_STORE, "not built"), (out, ops.EPILOGUE_STORE, "not built")):
        with pytest.raises(ops.KernelError, match=what):
            ops.gemm_q8_debug(out_[:, :128], a, sa, w[:128], sw[:128], epilogue, status, 4096, 1)
    b, sb, v, sv = _operands(17, 128, 256, 2)
    with pytest.raises(ops.KernelError, match="16 tokens"):
        ops.gemm_q8_debug(torch.zeros(17, 128, device=DEV), b, sb, v, sv, ops.EPILOGUE_ACCUMULATE, status, 4096, 1)
    for limit, block, what in ((4096, 1, "at most 8 CTAs"), (0, 1, "wait_limit"), (1 << 17, 1, "wait_limit"), (4096, 2, "no block"), (4096, -1, "no block")):
        with pytest.raises(ops.KernelError, match=what):
            ops.gemm_q8_debug(out, a, sa, w, sw, ops.EPILOGUE_ACCUMULATE, status, limit, block)
    assert not out.any() and status.tolist() == [0, 0, 0, 0]
