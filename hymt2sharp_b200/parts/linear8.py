"""A weight matrix in 8-bit integers with a scale for each output channel, and the rows of 8-bit integers that it multiplies.

A Linear8 stands where a Linear stands.  It quantises the stored weights once, when it is made; what it is called with becomes 8-bit rows with a scale
for each token, unless it is such rows already (a norm makes them on its way: RMSNorm.rows8).  Sums are exact; the scales are applied in float32
(kernels.ops.gemm_q8_tc)."""
from __future__ import annotations

from dataclasses import dataclass

import torch

from ..kernels import ops
from .linear import Linear, compute_form

WEIGHT_KINDS = (None, "int8")     # as the checkpoint stores them (None), or 8-bit integers


@dataclass
class Rows8:
    """Rows of 8-bit integers [T, dim] with a float32 scale each."""
    q: torch.Tensor
    scale: torch.Tensor

    @property
    def shape(self):
        return self.q.shape

    @property
    def device(self):
        return self.q.device

    @staticmethod
    def room(rows: int, width: int, device) -> "Rows8":
        return Rows8(ops.q8_rows(rows, width, device), torch.empty(rows, dtype=torch.float32, device=device))

    @staticmethod
    def of(x: torch.Tensor) -> "Rows8":
        rows = Rows8.room(*x.shape, x.device)
        ops.quantize_q8(rows.q, rows.scale, x)
        return rows

    def values(self, dtype: torch.dtype) -> torch.Tensor:
        """What the rows stand for."""
        out = torch.empty(self.q.shape, dtype=dtype, device=self.q.device)
        ops.dequantize_q8(out, self.q, self.scale)
        return out


class Linear8:
    """y = epilogue(x @ W^T) with W in 8-bit integers [out, in] and a scale a row; epilogue, role, glu and glu_bias as for Linear.  `dtype` is what
    its outputs have where the call does not say (its inputs may be 8-bit rows, which have none).  `settled`: whoever made the weights has waited for them and
    leaves them as they are, so that a product may fetch them while the kernel in front of it runs; without it they may come from that very kernel."""

    def __init__(self, weight: Rows8, dtype: torch.dtype, epilogue: int = ops.EPILOGUE_STORE, role: str | None = None, glu: "ops.GluRule | None" = None,
                 glu_bias: torch.Tensor | None = None, settled: bool = False):
        self.rows, self.dtype, self.settled = weight, dtype, settled
        self.weight, self.scale = weight.q, weight.scale
        self.epilogue, self.role, self.glu, self.glu_bias = epilogue, role, glu, glu_bias
        self.out_features = weight.shape[0] // 2 if epilogue == ops.EPILOGUE_SWIGLU else weight.shape[0]
        self.in_features = weight.shape[1]

    def __call__(self, x, out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None, ctx=None) -> torch.Tensor:
        """x: activations, or Rows8."""
        ops.tag = self.role
        try:
            rows = x if isinstance(x, Rows8) else Rows8.of(x if x.stride(-1) == 1 else x.contiguous())
            if out is None:
                out = torch.empty((x.shape[0], self.out_features), dtype=out_dtype or self.dtype, device=x.device)
            ops.gemm_q8_tc(out, rows.q, rows.scale, self.weight, self.scale, self.epilogue, ops.device_status(out.device), self.glu, self.glu_bias,
                           weights_settled=self.settled)
        finally:
            ops.tag = None
        return out

    def add_then_norm(self, x, residual: torch.Tensor, norm, ctx) -> None:
        """residual += x @ W^T; the norm behind it runs by itself (it makes the next product's 8-bit rows)."""
        if ctx is not None:
            ctx.prenormed = None
        self(x, out=residual)


def make_linear(weights: str | None, weight: torch.Tensor, device, dtype: torch.dtype, epilogue: int = ops.EPILOGUE_STORE, **more):
    """The product with a stored matrix: as it is stored (`weights` None) or in 8-bit integers ("int8")."""
    check_weights(weights)
    if weights is None:
        return Linear(compute_form(weight, device, dtype), epilogue, **more)
    rows = Rows8.of(weight.to(device).contiguous())
    torch.cuda.current_stream(rows.device).synchronize()      # (every later product may fetch them before the kernel in front of it is through)
    return Linear8(rows, dtype, epilogue, settled=True, **more)


def same_weight(linear, epilogue: int):
    """Another product with the matrix of `linear`."""
    if isinstance(linear, Linear8):
        return Linear8(linear.rows, linear.dtype, epilogue, role=linear.role, settled=linear.settled)
    return Linear(linear.weight, epilogue, role=linear.role)


def check_weights(weights: str | None) -> None:
    if weights not in WEIGHT_KINDS:
        raise ValueError(f"weights '{weights}' are not known (known: {', '.join(str(k) for k in WEIGHT_KINDS)})")
