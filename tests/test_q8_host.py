"""What the operators on 8-bit rows refuse, before anything is launched (no GPU: tensors on the CPU are themselves the last thing refused)."""
import pytest
import torch

from hymt2sharp_b200.kernels import ops

BF, F32 = torch.bfloat16, torch.float32


def _rows(rows, width):
    return ops.q8_rows(rows, width, "cpu"), torch.empty(rows)


@pytest.mark.parametrize("rows, width", [(1, 1), (3, 15), (3, 16), (5, 17), (0, 40)])
def test_rows_start_on_16_bytes(rows, width):
    q = ops.q8_rows(rows, width, "cpu")
    assert q.shape == (rows, width) and q.stride(1) == 1 and q.stride(0) % 16 == 0 and 0 <= q.stride(0) - width < 16


def test_what_is_fine_but_for_its_device():
    q, s = _rows(3, 40)
    w, ws = _rows(6, 40)
    status = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: ops.quantize_q8(q, s, torch.empty(3, 40)), lambda: ops.dequantize_q8(torch.empty(3, 40), q, s),
                 lambda: ops.rmsnorm_q8(q, s, torch.empty(3, 40), torch.empty(40), 1e-5),
                 lambda: ops.gemm_q8_tc(torch.empty(3, 6), q, s, w, ws, ops.EPILOGUE_STORE, status)):
        with pytest.raises(ops.KernelError, match="current CUDA device"):
            call()


@pytest.mark.parametrize("q, s, x, what", [
    (torch.empty(3, 32), torch.empty(3), torch.empty(3, 32), "int8 matrix"),
    (torch.empty(3, 40, dtype=torch.int8), torch.empty(3), torch.empty(3, 40), "start on 16 bytes"),       # rows 40 bytes apart
    (torch.empty(48, 3, dtype=torch.int8).t(), torch.empty(3), torch.empty(3, 48), "start on 16 bytes"),
    (torch.empty(32, dtype=torch.int8).expand(3, 32), torch.empty(3), torch.empty(3, 32), "start on 16 bytes"),
    (torch.empty(3, 64, dtype=torch.int8)[:, 8:40], torch.empty(3), torch.empty(3, 32), "start on 16 bytes"),
    (torch.empty(3, 32, dtype=torch.int8), torch.empty(2), torch.empty(3, 32), "3 rows need as many"),
    (torch.empty(3, 32, dtype=torch.int8), torch.empty(3, dtype=BF), torch.empty(3, 32), "3 rows need as many"),
    (torch.empty(3, 32, dtype=torch.int8), torch.empty(6)[::2], torch.empty(3, 32), "3 rows need as many"),
    (torch.empty(3, 32, dtype=torch.int8), torch.empty(3), torch.empty(3, 31), r"\(3, 32\)|\[3, 32\]"),
    (torch.empty(3, 32, dtype=torch.int8), torch.empty(3), torch.empty(32, 3).t(), "contiguous rows"),
    (torch.empty(3, 32, dtype=torch.int8), torch.empty(3), torch.empty(32).expand(3, 32), "contiguous rows"),
    (torch.empty(3, 32, dtype=torch.int8), torch.empty(3), torch.empty(3, 32, dtype=torch.float16), "not supported"),
    (torch.empty(3, 0, dtype=torch.int8), torch.empty(3), torch.empty(3, 0), "without entries")])
def test_rows_that_are_not_taken(q, s, x, what):
    if q.data_ptr() % 16 == 0 and x.shape[1] == 0:
        q = torch.empty(3, 16, dtype=torch.int8)[:, :0]
    with pytest.raises(ops.KernelError, match=what):
        ops.quantize_q8(q, s, x)
    with pytest.raises(ops.KernelError, match=what):
        ops.rmsnorm_q8(q, s, x, torch.empty(q.shape[1]), 1e-5)
    if what != "without entries":
        with pytest.raises(ops.KernelError, match=what):
            ops.dequantize_q8(x, q, s)


def test_norms_that_are_not_taken():
    q, s = _rows(3, 32)
    x, g = torch.empty(3, 32), torch.empty(32)
    for change, what in ((dict(gain=torch.empty(31)), "gain"), (dict(gain=torch.empty(64)[::2]), "gain"), (dict(gain=g.half()), "not supported"),
                         (dict(add=torch.empty(2, 32)), "add"), (dict(add=x.half()), "not supported"), (dict(total=x), "total"),
                         (dict(add=x, total=x.bfloat16()), "total"), (dict(add=x, total=torch.empty(3, 33)), "total")):
        with pytest.raises(ops.KernelError, match=what):
            ops.rmsnorm_q8(**{**dict(q=q, scale=s, x=x, gain=g, eps=1e-5), **change})


def test_products_that_are_not_taken():
    a, sa = _rows(3, 32)
    w, sw = _rows(6, 32)
    ok = dict(out=torch.empty(3, 6), a=a, a_scale=sa, w=w, w_scale=sw, epilogue=ops.EPILOGUE_STORE, status=torch.zeros(4, dtype=torch.int32))
    long_a, long_w = ops.q8_rows(1, ops.Q8_MAX_INNER + 1, "cpu"), ops.q8_rows(2, ops.Q8_MAX_INNER + 1, "cpu")
    for change, what in ((dict(w=ops.q8_rows(6, 31, "cpu")), "do not go together"), (dict(out=torch.empty(3, 5)), "out"),
                         (dict(a=torch.empty(3, 32)), "a must be an int8"), (dict(w=torch.empty(6, 33, dtype=torch.int8)), "16 bytes"),
                         (dict(w_scale=torch.empty(7)), "6 rows"), (dict(a_scale=torch.empty(1)), "3 rows"),
                         (dict(out=torch.empty(3, 6, dtype=BF), epilogue=ops.EPILOGUE_ACCUMULATE), "not built"), (dict(epilogue=7), "not built"),
                         (dict(out=torch.empty(3, 2), w=ops.q8_rows(5, 32, "cpu"), w_scale=torch.empty(5), epilogue=ops.EPILOGUE_SWIGLU), "do not go together"),
                         (dict(out=torch.empty(3, 6, dtype=torch.float16)), "not supported"), (dict(status=torch.zeros(4)), "status"),
                         (dict(out=torch.empty(6).expand(3, 6)), "contiguous rows"),
                         (dict(out=torch.empty(1, 2), a=long_a, a_scale=torch.empty(1), w=long_w, w_scale=torch.empty(2)), "do not go together")):
        with pytest.raises(ops.KernelError, match=what):
            ops.gemm_q8_tc(**{**ok, **change})


@pytest.mark.parametrize("gated", [False, True])
def test_plans_stay_within_the_machine(gated):
    """Shared memory, tensor memory, clusters and the cover of K, over the range of sizes; nothing is launched."""
    from hymt2sharp_b200.kernels import build
    try:
        build.find_nvcc()
    except build.BuildError as err:
        pytest.skip(str(err))
    sizes = [1, 2, 15, 16, 17, 33, 64, 65, 100, 128, 129, 200, 257, 500, 512, 513, 1000, 4096, 30000]
    for T in sizes + [200000]:
        for N in [1, 100, 128, 129, 500, 2048, 6144, 28672, 152064]:
            for K in [1, 64, 128, 129, 500, 2048, 14336, ops.Q8_MAX_INNER]:
                for sms in (148, 132):
                    p = ops.gemm_q8_describe(T, N, K, gated, sms)
                    blocks, accs = -(-K // 128), 2 if gated else 1
                    assert 2 <= p["stages"] <= 12 and 1 <= p["splits"] <= 8
                    assert p["splits"] * p["k_blocks"] >= blocks > (p["splits"] - 1) * p["k_blocks"]
                    if p["few"]:
                        assert T <= 512 and p["width"] in (16, 32, 64, 128) and accs * p["width"] <= 256
                        stage, sums = accs * 16384 + p["width"] * 128, accs * p["width"] * 512
                        assert p["shared_bytes"] >= max(p["stages"] * stage, sums) + 1024 and p["shared_bytes"] <= 226 * 1024
                        assert p["ctas"] == -(-N // 128) * -(-T // p["width"]) * p["splits"]
                    else:
                        assert T > 64 and p["splits"] == 1 and 64 <= p["width"] <= 256 and p["width"] % (64 if gated else 32) == 0 and p["ctas"] % 2 == 0 and 2 <= p["ctas"] <= sms
                        assert p["stages"] * (16384 + p["width"] * 64) + 32768 + 1024 == p["shared_bytes"] <= 226 * 1024


@pytest.mark.parametrize("rows,width", [(1, ops.Q8_MOST + 1), (ops.Q8_MOST + 1, 1)])
def test_matrices_beyond_what_is_counted(rows, width):
    q = torch.empty_strided((rows, width), ((width + 15) & ~15, 1), dtype=torch.int8, device="meta")
    s, x = torch.empty(rows, device="meta"), torch.empty(rows, width, device="meta")
    for call in (lambda: ops.quantize_q8(q, s, x), lambda: ops.dequantize_q8(x, q, s), lambda: ops.rmsnorm_q8(q, s, x, torch.empty(width, device="meta"), 1e-5)):
        with pytest.raises(ops.KernelError, match="at most"):
            call()
