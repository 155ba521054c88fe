"""What a product with 8-bit weights tells its kernel about them (no GPU: the kernels are stood in for)."""
import pytest
import torch

from hymt2sharp_b200.kernels import ops
from hymt2sharp_b200.parts import Linear8, Rows8
from hymt2sharp_b200.parts.linear8 import make_linear, same_weight


@pytest.fixture
def calls(monkeypatch):
    """The order of the launches that the parts ask for, with what a product says about its weights."""
    made = []

    class Stream:
        def synchronize(self):
            made.append("wait")
    monkeypatch.setattr(ops, "quantize_q8", lambda q, scale, x: made.append("rows"))
    monkeypatch.setattr(ops, "gemm_q8_tc", lambda *args, weights_settled=False: made.append(("product", weights_settled)))
    monkeypatch.setattr(ops, "device_status", lambda device: None)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream())
    return made


def test_weights_that_nobody_waited_for_are_not_fetched_ahead(calls):
    """Rows that were there before, then a weight matrix that becomes integers, then their product: the kernel in front of the product makes its weights."""
    x = Rows8.of(torch.randn(3, 32))
    linear = Linear8(Rows8.of(torch.randn(6, 32)), torch.float32)
    linear(x)
    same_weight(linear, ops.EPILOGUE_ACCUMULATE)(x, out=torch.empty(3, 6))
    assert calls == ["rows", "rows", ("product", False), ("product", False)]


def test_a_models_weights_are_waited_for_once_and_fetched_ahead(calls):
    linear = make_linear("int8", torch.randn(6, 32), torch.device("cpu"), torch.float32)
    assert calls == ["rows", "wait"]
    linear(torch.randn(3, 32))
    same_weight(linear, ops.EPILOGUE_ACCUMULATE)(torch.randn(3, 32), out=torch.empty(3, 6))
    assert calls[2:] == ["rows", ("product", True)] * 2
