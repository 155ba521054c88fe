"""Gated products of 8-bit integers into float32: the gate's function is off by a few roundings of float32, however far the gate lies from zero."""
import pytest
import torch

from test_gpu_kernels import DEV, _ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24                                     # half a step of float32, relative


@pytest.mark.parametrize("T", [3, 40, 100, 300])
@pytest.mark.parametrize("rule", [None, (60.0, 1.702)])
def test_float32_gates(T, rule):
    """Sums and scales whose products are exact, so that the gate's function alone is seen: gates of -64 to 63.5, ups of 1 (clamped: 1 + 1)."""
    ops = _ops()
    N, K = 256, 16
    a, w = ops.q8_rows(T, K, DEV), ops.q8_rows(2 * N, K, DEV)
    a.zero_(), w.zero_()
    a[:, 0] = 1
    w[:N, 0] = torch.arange(-128, 128, device=DEV).to(torch.int8)
    w[N:, 0] = 4
    sa = torch.ones(T, device=DEV)
    sa[1::2] = 0.25
    sw = torch.cat([torch.full((N,), 0.5, device=DEV), torch.full((N,), 0.25, device=DEV)])
    status = torch.zeros(4, dtype=torch.int32, device=DEV)
    out = torch.empty(T, N, device=DEV)
    ops.gemm_q8_tc(out, a, sa, w, sw, ops.EPILOGUE_SWIGLU, status, glu=None if rule is None else ops.GluRule("clamped", *rule))
    y = (a.double() @ w.double().T) * sa.double()[:, None] * sw.double()
    g, u = y[:, :N], y[:, N:]
    alpha = 1.0
    if rule is not None:
        g, u, alpha = g.clamp(max=rule[0]), u.clamp(-rule[0], rule[0]) + 1, rule[1]
    want = g / (1 + torch.exp(-alpha * g)) * u
    # the exponential within two steps of its result (4 U), its argument's rounding (none where alpha is 1; alpha itself is a float32), the addition, the reciprocal
    # within a step (2 U) and the product with the gate; that with u + 1 is exact here
    bound = (8 * U + (0 if rule is None else 2 * U * (alpha * g).abs())) * 1.01 * want.abs()
    # float32 has no e^x beyond x = 88.72, where e^-x = 2.96e-39: the sum is infinite there and the result 0, in place of at most 64 e^-88.72 (1 + 1) = 3.8e-37.
    # From e^87.33 = 2^126 on the reciprocal has no leading one any more: a whole number of 2^-149, times the same 128 below 1e-42
    bound = bound + torch.where(-alpha * g > 87.3, 3.9e-37, 0.0)
    assert ((out.double() - want).abs() <= bound).all()
    assert status.tolist() == [0, 0, 0, 0]
