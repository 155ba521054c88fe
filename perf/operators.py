"""The operators of dense layers with 8-bit integer weights and activations, as they are timed: rows that become 8-bit integers with a scale
each (and are read back), RMSNorm with the residual's addition in front and 8-bit rows behind, and the product of 8-bit rows with 8-bit weights,
which has a scale for each token and one for each output channel; and the three together as a gated feed-forward.

`listed()` names the cases, `draw(rng)` gives more of the same ranges, `prepare` makes what a program holds before the call, `run` makes one
pass (in elementary torch operations, or with `own` by the framework's kernels), `exact` says in 64 bits what that pass computes.

A row x becomes integers q and a scale s:  q = 127 x / max|x| rounded to the nearest whole number (ties to even),  s = max|x| / 127;  it stands
for q s.  A row that holds a NaN or an infinity has the scale NaN and zeros.  Norm:  t = x + add in x's type,  r = 1 / sqrt(mean(t^2) + eps);
what becomes integers is t gain in float32, and r, which is the same for the whole row, goes into the scale.
Product:  y[t, n] = a_scale[t] w_scale[n] sum_k a[t, k] w[n, k].
"""
from __future__ import annotations

import math
import random

import torch

own = False                    # False: elementary torch operations; True: the framework's kernels
ops = None                     # the framework's operators, imported by the first pass that calls them

DEV = "cuda:0"
EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
OUTLIERS = 0.004               # share of the channels that are larger than the others, as activations of language models have them
LIMIT, ALPHA = 7.0, 1.702      # of the clamped gate


def _gemm(name, rows, out, inner, epilogue="store", dtype="bf16", glu="silu"):
    return dict(name=name, kind="gemm", rows=rows, out=out, inner=inner, epilogue=epilogue, dtype=dtype, glu=glu)


def _norm(name, rows, width, dtype="f32", add="bf16"):
    return dict(name=name, kind="norm", rows=rows, width=width, dtype=dtype, add=add)


def _rows(name, rows, width, dtype="bf16"):
    return dict(name=name, kind="rows", rows=rows, width=width, dtype=dtype)


def listed() -> list:
    return [
        # one token of a chat through an output projection: the smallest call, launch and memory latency
        _gemm("gemm_1_token", 1, 2048, 2048),
        # a decode step of a small batch through the gate and up projections of the 7B-family sizes: the weights' bytes
        _gemm("gemm_gated_8", 8, 14336, 4096, "gated"),
        # a decode step of a larger batch into the residual rows, an odd number of sequences
        _gemm("gemm_add_61", 61, 4096, 14336, "add", "f32"),
        # a prompt of odd length through sizes that no tile divides, a clamped gate with biases
        _gemm("gemm_odd_531", 531, 1021, 1111, "gated", "f32", "clamped"),
        # a prompt through the query, key and value projection of the 7B-family sizes
        _gemm("gemm_2048", 2048, 6144, 4096),
        # a batch of long prompts through its gate and up projections: the largest work
        _gemm("gemm_gated_8192", 8192, 14336, 4096, "gated"),
        # the norm of a decode step: two rows, the attention's output joins the residual
        _norm("norm_2", 2, 4096),
        # the norm of a batch of prompts
        _norm("norm_8192", 8192, 4096),
        # rows of an odd width in 16 bits, nothing added
        _norm("norm_odd_1777", 1777, 1531, "bf16", "none"),
        # a decode step's activations in front of the down projection
        _rows("rows_16", 16, 14336),
        # and a prompt's
        _rows("rows_8192", 8192, 14336),
        # norm, gate and up, 8-bit rows, down: a feed-forward of the 1.8B sizes on a prompt of odd length
        dict(name="ffn_1777", kind="ffn", rows=1777, hidden=2048, inner=6144),
    ]


LARGEST = 8192 * 28672 * 4096  # multiply-adds of the largest listed product
MOST_ENTRIES = 8192 * 14336


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["gemm", "gemm", "gemm", "norm", "norm", "rows", "rows", "ffn"])
    if kind == "gemm":
        epilogue = rng.choice(["store", "add", "gated"])
        out, inner = _log_int(rng, 64, 16384), _log_int(rng, 64, 16384)
        if rng.random() < 0.5:          # (half of them the multiples that models have, half any number)
            out, inner = -(-out // 64) * 64, -(-inner // 64) * 64
        most = LARGEST // (out * inner * (2 if epilogue == "gated" else 1))
        c = _gemm("", _log_int(rng, 1, min(8192, most)), out, inner, epilogue, "f32" if epilogue == "add" else rng.choice(["bf16", "bf16", "f32"]),
                  rng.choice(["silu", "silu", "clamped"]) if epilogue == "gated" else "silu")
    elif kind == "ffn":
        hidden = rng.choice([1024, 2048, 4096, rng.randint(64, 4096)])
        inner = _log_int(rng, 64, 14336)
        c = dict(kind="ffn", rows=_log_int(rng, 1, 4096), hidden=hidden, inner=inner)
    else:
        width = _log_int(rng, 1, 16384 if kind == "norm" else 28672)
        if rng.random() < 0.5:
            width = -(-width // 64) * 64
        rows = _log_int(rng, 1, max(1, min(16384, MOST_ENTRIES // (2 * width))))
        c = _norm("", rows, width, rng.choice(["f32", "bf16"]), rng.choice(["none", "bf16", "f32"])) if kind == "norm" \
            else _rows("", rows, width, rng.choice(["bf16", "f32"]))
    c.pop("name", None)
    return c


# -- inputs ------------------------------------------------------------------------------------------------------------------
def _activations(gen, rows, width, dtype, scale=1.0):
    """Normal entries, each row and some channels of a size of their own."""
    x = torch.randn(rows, width, generator=gen, device=DEV)
    x *= torch.exp(0.3 * torch.randn(rows, 1, generator=gen, device=DEV)) * scale
    channels = torch.rand(width, generator=gen, device=DEV) < OUTLIERS
    x *= torch.where(channels, 12.0, 1.0)
    return x.to(dtype)


def _codes(pieces, rows, width):
    """(q, s) of float32 rows that come in pieces, as the 8-bit kernels keep them: a row of q starts on a multiple of 16 bytes."""
    q = torch.zeros(rows, -(-width // 16) * 16, dtype=torch.int8, device=DEV)[:, :width]
    s = torch.empty(rows, dtype=torch.float32, device=DEV)
    at = 0
    for x in pieces:
        here = slice(at, at + x.shape[0])
        s[here] = x.abs().amax(1) / 127.0
        q[here] = torch.round(x / s[here, None]).clamp(-127, 127)
        at += x.shape[0]
    return q, s


def _weights(gen, rows, inner):
    """A weight matrix's integers and scales; made in pieces, so that a large one's float32 form is never held whole."""
    return _codes((torch.randn(min(4096, rows - r), inner, generator=gen, device=DEV) / math.sqrt(inner) for r in range(0, rows, 4096)), rows, inner)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed) * 7919 + 17)
    kind, st = case["kind"], {"case": case}
    if kind == "gemm":
        dtype, gated = TYPES[case["dtype"]], case["epilogue"] == "gated"
        st["a"], st["a_scale"] = _codes([_activations(gen, case["rows"], case["inner"], torch.float32)], case["rows"], case["inner"])
        st["w"], st["w_scale"] = _weights(gen, case["out"] * (2 if gated else 1), case["inner"])
        if case["epilogue"] == "add":
            st["residual"] = torch.randn(case["rows"], case["out"], generator=gen, device=DEV, dtype=dtype)
        if gated and case["glu"] == "clamped":
            st["bias"] = torch.randn(2 * case["out"], generator=gen, device=DEV)
    elif kind == "norm":
        st["x"] = _activations(gen, case["rows"], case["width"], TYPES[case["dtype"]], 2.0)
        if case["add"] != "none":
            st["add"] = _activations(gen, case["rows"], case["width"], TYPES[case["add"]])
        st["gain"] = (1.0 + 0.1 * torch.randn(case["width"], generator=gen, device=DEV)).to(torch.bfloat16)
    elif kind == "rows":
        st["x"] = _activations(gen, case["rows"], case["width"], TYPES[case["dtype"]])
    else:
        st["x"] = _activations(gen, case["rows"], case["hidden"], torch.float32, 2.0)
        st["add"] = _activations(gen, case["rows"], case["hidden"], torch.bfloat16)
        st["gain"] = (1.0 + 0.1 * torch.randn(case["hidden"], generator=gen, device=DEV)).to(torch.bfloat16)
        st["w_in"], st["w_in_scale"] = _weights(gen, 2 * case["inner"], case["hidden"])
        st["w_down"], st["w_down_scale"] = _weights(gen, case["hidden"], case["inner"])
    return st


# -- the plain form -----------------------------------------------------------------------------------------------------------
def _plain_codes(x):
    """float32 rows -> (whole numbers as float32, scales); in 64 bits, for the entries half way between two whole numbers."""
    top = x.abs().amax(1).double()
    q = torch.round(x.double() * 127.0 / top[:, None])
    return torch.nan_to_num(q, 0.0, 0.0, 0.0).float(), torch.where(torch.isfinite(top), top / 127.0, torch.nan).float()


def _plain_norm(x, add, gain):
    t = x.float() if add is None else x.float() + add.float()
    t = t.to(x.dtype)              # the rows as they are kept
    r = torch.rsqrt(t.float().pow(2).mean(1) + EPS)
    q, s = _plain_codes(t.float() * gain.float())
    return t, q, s * r


def _plain_glu(g, u, glu):
    if glu == "silu":
        return g / (1.0 + torch.exp(-g)) * u
    g, u = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
    return g / (1.0 + torch.exp(-ALPHA * g)) * (u + 1.0)


def _plain_product(a, a_scale, w, w_scale):
    return (a.float() @ w.float().t()) * a_scale[:, None] * w_scale[None, :]


def _plain(st):
    case = st["case"]
    if case["kind"] == "gemm":
        y, n = _plain_product(st["a"], st["a_scale"], st["w"], st["w_scale"]), case["out"]
        if case["epilogue"] == "add":
            y = st["residual"] + y
        elif case["epilogue"] == "gated":
            if "bias" in st:
                y = y + st["bias"]
            y = _plain_glu(y[:, :n], y[:, n:], case["glu"])
        return {"y": y.to(TYPES[case["dtype"]])}
    if case["kind"] == "norm":
        t, q, s = _plain_norm(st["x"], st.get("add"), st["gain"])
        out = {"values": q * s[:, None], "scale": s}
        if "add" in st:
            out["total"] = t
        return out
    if case["kind"] == "rows":
        q, s = _plain_codes(st["x"].float())
        return {"values": q * s[:, None], "scale": s}
    t, q, s = _plain_norm(st["x"], st["add"], st["gain"])
    y = _plain_product(q, s, st["w_in"], st["w_in_scale"])
    q, s = _plain_codes(_plain_glu(y[:, :case["inner"]], y[:, case["inner"]:], "silu").to(torch.bfloat16).float())
    return {"total": t, "y": _plain_product(q, s, st["w_down"], st["w_down_scale"]).to(torch.bfloat16)}


# -- the framework's calls ------------------------------------------------------------------------------------------------------
def _scales(rows):
    return torch.empty(rows, dtype=torch.float32, device=DEV)


def _own_norm(st, rows, width):
    q, s = ops.q8_rows(rows, width, DEV), _scales(rows)
    total = torch.empty_like(st["x"]) if "add" in st else None
    ops.rmsnorm_q8(q, s, st["x"], st["gain"], EPS, add=st.get("add"), total=total)
    return total, q, s


def _own_values(q, s):
    values = torch.empty(q.shape, dtype=torch.float32, device=DEV)
    ops.dequantize_q8(values, q, s)
    return values


def _own(st):
    case, status = st["case"], ops.device_status(DEV)
    rows = case["rows"]
    if case["kind"] == "gemm":
        if case["epilogue"] == "add":
            y = st["residual"].clone()             # (the call adds in place)
            ops.gemm_q8_tc(y, st["a"], st["a_scale"], st["w"], st["w_scale"], ops.EPILOGUE_ACCUMULATE, status)
            return {"y": y}
        y = torch.empty(rows, case["out"], dtype=TYPES[case["dtype"]], device=DEV)
        if case["epilogue"] == "store":
            ops.gemm_q8_tc(y, st["a"], st["a_scale"], st["w"], st["w_scale"], ops.EPILOGUE_STORE, status)
        else:
            rule = None if case["glu"] == "silu" else ops.GluRule("clamped", LIMIT, ALPHA)
            ops.gemm_q8_tc(y, st["a"], st["a_scale"], st["w"], st["w_scale"], ops.EPILOGUE_SWIGLU, status, glu=rule, glu_bias=st.get("bias"))
        return {"y": y}
    if case["kind"] == "norm":
        total, q, s = _own_norm(st, rows, case["width"])
        out = {"values": _own_values(q, s), "scale": s}
        if total is not None:
            out["total"] = total
        return out
    if case["kind"] == "rows":
        q, s = ops.q8_rows(rows, case["width"], DEV), _scales(rows)
        ops.quantize_q8(q, s, st["x"])
        return {"values": _own_values(q, s), "scale": s}
    total, q, s = _own_norm(st, rows, case["hidden"])
    act = torch.empty(rows, case["inner"], dtype=torch.bfloat16, device=DEV)
    ops.gemm_q8_tc(act, q, s, st["w_in"], st["w_in_scale"], ops.EPILOGUE_SWIGLU, status)
    q, s = ops.q8_rows(rows, case["inner"], DEV), _scales(rows)
    ops.quantize_q8(q, s, act)
    y = torch.empty(rows, case["hidden"], dtype=torch.bfloat16, device=DEV)
    ops.gemm_q8_tc(y, q, s, st["w_down"], st["w_down_scale"], ops.EPILOGUE_STORE, status)
    return {"total": total, "y": y}


def run(state):
    global ops
    if own:
        if ops is None:
            from hymt2sharp_b200.kernels import ops
        return _own(state)
    return _plain(state)


# -- what a pass cannot do without ---------------------------------------------------------------------------------------------
def work(case) -> dict:
    size = {"bf16": 2, "f32": 4, "none": 0}
    rows = case["rows"]
    if case["kind"] == "gemm":
        n, k, b = case["out"] * (2 if case["epilogue"] == "gated" else 1), case["inner"], size[case["dtype"]]
        read = rows * k + n * k + 4 * (rows + n) + (4 * n if case["glu"] == "clamped" else 0) + (rows * case["out"] * b if case["epilogue"] == "add" else 0)
        return {"bytes": read + rows * case["out"] * b, "flops": 2.0 * rows * n * k}
    if case["kind"] == "ffn":
        h, f = case["hidden"], case["inner"]
        return {"bytes": rows * h * (4 + 2 + 4 + 2) + 3 * h * f + 4 * (2 * f + h) + 2 * h, "flops": 6.0 * rows * h * f}
    entries = rows * case["width"]
    if case["kind"] == "norm":     # (the 8-bit rows are written, and so are the values that they stand for)
        add = size[case["add"]]
        moved = entries * (size[case["dtype"]] + add + (size[case["dtype"]] if add else 0) + 1 + 4) + 4 * rows + 2 * case["width"]
        return {"bytes": moved, "flops": 8.0 * entries}
    return {"bytes": entries * (size[case["dtype"]] + 1 + 4) + 4 * rows, "flops": 5.0 * entries}


# -- 64 bits -------------------------------------------------------------------------------------------------------------------
def _codes64(x):
    top = x.abs().max(dim=1, keepdim=True).values
    s = top / 127
    q = torch.where(top > 0, torch.round(127 * x / top), torch.zeros_like(x))
    return q, s


def _gate64(g, u, clamped):
    if clamped:
        g, u = torch.minimum(g, torch.full_like(g, LIMIT)), u.clamp(-LIMIT, LIMIT)
        return g * torch.sigmoid(ALPHA * g) * (u + 1)
    return g * torch.sigmoid(g) * u


def exact(case, seed):
    st = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    if case["kind"] == "gemm":
        y = torch.einsum("tk,nk->tn", st["a"], st["w"]) * torch.outer(st["a_scale"], st["w_scale"])
        if case["epilogue"] == "add":
            y += st["residual"]
        if case["epilogue"] == "gated":
            g, u = (y + st.get("bias", 0.0)).chunk(2, dim=1)
            y = _gate64(g, u, case["glu"] == "clamped")
        return {"y": y}
    if case["kind"] == "rows":
        q, s = _codes64(st["x"])
        return {"values": q * s, "scale": s[:, 0]}
    total = st["x"] + st["add"] if "add" in st else st["x"]
    kept = total.to(torch.bfloat16).double() if case.get("dtype") == "bf16" else total.float().double()       # the rows as they are kept
    q, s = _codes64((kept * st["gain"]).float().double())
    s = s / torch.sqrt((kept * kept).mean(dim=1, keepdim=True) + EPS)
    if case["kind"] == "norm":
        out = {"values": q * s, "scale": s[:, 0]}
        if "add" in st:
            out["total"] = total
        return out
    g, u = (torch.einsum("tk,nk->tn", q * s, st["w_in"]) * st["w_in_scale"]).chunk(2, dim=1)
    q, s = _codes64(_gate64(g, u, False).to(torch.bfloat16).double())
    return {"total": total, "y": torch.einsum("tk,nk->tn", q * s, st["w_down"]) * st["w_down_scale"]}
