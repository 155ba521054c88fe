"""A block with 8-bit weights whose gate is clamped or has biases: a prompt's step launched by one call against the same kernels one by one, and against the block
with the matrices that the integers stand for."""
from dataclasses import replace

import pytest
import torch

from test_gpu_kernels import DEV, _ops

pytestmark = pytest.mark.gpu

BIASES = dict(gate_bias="gb", up_bias="ub")


def _rounded(x):
    """What the 8-bit rows of x stand for."""
    top = x.abs().amax(-1, keepdim=True)
    return torch.nan_to_num(torch.round(127 * x / top)) * top / 127


def _block(d, hidden, inner, kind, more, weights):
    from hymt2sharp_b200.parts.base import PartSpec, build_part
    norm = lambda n: PartSpec("rmsnorm", dict(dim=hidden, eps=1e-5, weight=n))
    attn = dict(hidden=hidden, heads=4, kv_heads=2, head_dim=d, eps=1e-5, qk_norm=True, position=None, q_proj="q", k_proj="k", v_proj="v", o_proj="o",
                q_norm="qn", k_norm="kn", weights=weights)
    ff = dict(hidden=hidden, intermediate=inner, gate_proj="g", up_proj="u", down_proj="d", weights=weights, **more)
    return build_part("block", PartSpec("pre_norm", dict(norm1=norm("n1"), mixer=PartSpec("gqa_attention", attn), norm2=norm("n2"), feed_forward=PartSpec(kind, ff))))


def _step(block, hidden, lens, twice=False):
    """The residual rows behind the block, of prompts of these lengths (with `twice`: and of a further piece of them)."""
    from hymt2sharp_b200.cache import PagedCache
    from hymt2sharp_b200.engine.engine import StepEntry, make_context
    from hymt2sharp_b200.parts.base import MixerSlot
    ops = _ops()
    dev = torch.device(DEV)
    cache = PagedCache([replace(block.cache_needs()[0], planes=1)], torch.bfloat16, dev, capacity_tokens=1024, block_tokens=64, max_slots=2, state_bytes=0)
    slots, outs, before = cache.alloc_slots(2), [], ops.launches
    g = torch.Generator(device=DEV).manual_seed(4)
    for _ in range(2 if twice else 1):
        ctx, _, _, plan = make_context(cache, [StepEntry(s, [0] * n) for s, n in zip(slots, lens)], 10, torch.bfloat16, dev, ops.device_status(dev))
        residual = torch.randn(sum(lens), hidden, generator=g, device=DEV)
        block.forward(residual, ctx, [MixerSlot(group=0, plane=0)])
        cache.end_step(plan)
        outs.append(residual)
    return torch.cat(outs), ops.launches - before


@pytest.mark.parametrize("d, hidden, inner", [(64, 96, 200), (128, 260, 203)])
@pytest.mark.parametrize("kind, more, one_call", [("clamped_glu", dict(limit=0.7, alpha=1.702), True), ("clamped_glu", dict(limit=0.7, alpha=1.702, **BIASES), True),
                                                  ("swiglu", BIASES, True), ("swiglu", dict(BIASES, down_bias="db"), False), ("swiglu", {}, True)])
def test_a_prompts_block_by_one_call(kind, more, one_call, d, hidden, inner, monkeypatch):
    ops = _ops()
    torch.manual_seed(3)
    small, wide = _block(d, hidden, inner, kind, more, "int8"), _block(d, hidden, inner, kind, more, None)
    stored = {n: torch.randn(s.shape) * (1 / s.shape[-1] ** 0.5 if len(s.shape) == 2 else 0.3) + (1.0 if s.init == "gain" else 0.0) for n, s in small.tensors().items()}
    stored = {n: w.bfloat16() if w.dim() == 2 or n in ("n1", "n2", "qn", "kn") else w for n, w in stored.items()}
    dev = torch.device(DEV)
    small.load(stored, dev, torch.bfloat16)
    calls, launch = [], ops.dense_block_q8
    monkeypatch.setattr(ops, "dense_block_q8", lambda *args: (calls.append(1), launch(*args)))
    whole, launches = _step(small, hidden, (40, 7), twice=True)
    assert len(calls) == (2 if one_call else 0)
    small.dense_rows8 = False
    parts, one_by_one = _step(small, hidden, (40, 7), twice=True)
    assert torch.equal(whole, parts) and launches == one_by_one and len(calls) == (2 if one_call else 0)
    wide.load({n: _rounded(w.double()).bfloat16() if w.dim() == 2 else w for n, w in stored.items()}, dev, torch.bfloat16)
    want, _ = _step(wide, hidden, (40, 7), twice=True)
    rms = ((whole - want).pow(2).mean() / want.pow(2).mean()).sqrt().item()
    # rows of integers: 0.9 % of a product, four of them one behind the other; 2^-9 for each of the roundings to bfloat16 (the weights', and some ten on the way)
    assert 0 < rms <= 4 * 0.009 + 0.002 * 11 ** 0.5, rms
    assert ops.device_status(dev).tolist() == [0, 0, 0, 0]


FORMS = [dict(value_dim=64), dict(norm_first=True), dict(sink=True), dict(head_gate="hg"), dict(q_bias="qb", k_bias="kb", v_bias="vb"),
         dict(qk_norm="all", norm_first=True), dict(own_kv=False), dict(window=9), dict(value_dim=64, norm_first=True, sink=True, head_gate="hg", q_bias="qb", k_bias="kb", v_bias="vb")]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("form", FORMS)
def test_attention_of_every_form(form, dtype):
    """Each form of grouped-query attention in a block with 8-bit weights, a prompt and a further piece of it, against the block with the matrices that the integers
    stand for.  (Without keys and values of its own: behind a block that has them, in the cache plane of that one.)"""
    from hymt2sharp_b200.cache import PagedCache
    from hymt2sharp_b200.engine.engine import StepEntry, make_context
    from hymt2sharp_b200.parts.base import MixerSlot, PartSpec, build_part
    ops = _ops()
    dev, hidden, d = torch.device(DEV), 96, 128

    def make(weights, form):
        norm = lambda n: PartSpec("rmsnorm", dict(dim=hidden, eps=1e-5, weight=n))
        attn = dict(dict(hidden=hidden, heads=4, kv_heads=2, head_dim=d, eps=1e-5, qk_norm=True, position=None, q_proj="q", k_proj="k", v_proj="v", o_proj="o",
                         q_norm="qn", k_norm="kn", weights=weights), **form)
        if not attn.get("own_kv", True):
            attn.update(k_proj=None, v_proj=None, k_norm=None)
        ff = dict(hidden=hidden, intermediate=200, gate_proj="g", up_proj="u", down_proj="d", weights=weights)
        return build_part("block", PartSpec("pre_norm", dict(norm1=norm("n1"), mixer=PartSpec("gqa_attention", attn), norm2=norm("n2"), feed_forward=PartSpec("swiglu", ff))))

    torch.manual_seed(5)
    alone = form.get("own_kv", True)
    blocks = [make("int8", form)] if alone else [make("int8", {}), make("int8", form)]
    plain = [make(None, form)] if alone else [make(None, {}), make(None, form)]
    outs = []
    stored = [{n: torch.randn(s.shape) * (1 / s.shape[-1] ** 0.5 if len(s.shape) == 2 else 0.1) + (1.0 if s.init == "gain" else 0.0) for n, s in b.tensors().items()}
              for b in blocks]
    if dtype == torch.bfloat16:
        stored = [{n: w.bfloat16() for n, w in of.items()} for of in stored]
    for set_, rounded in ((blocks, False), (plain, True)):
        for b, of in zip(set_, stored):
            b.load({n: _rounded(w.double()).to(w.dtype) if rounded and w.dim() == 2 else w for n, w in of.items()}, dev, dtype)
        cache = PagedCache([replace(set_[0].cache_needs()[0], planes=1)], dtype, dev, capacity_tokens=256, block_tokens=64, max_slots=2, state_bytes=0)
        slots = cache.alloc_slots(2)
        g = torch.Generator(device=DEV).manual_seed(6)
        rows = []
        for lens in ((40, 7), (1, 1), (3, 20)):
            ctx, _, _, plan = make_context(cache, [StepEntry(s, [0] * n) for s, n in zip(slots, lens)], 10, dtype, dev, ops.device_status(dev))
            residual = torch.randn(sum(lens), hidden, generator=g, device=DEV)
            for i, b in enumerate(set_):
                b.forward(residual, ctx, [MixerSlot(group=0, plane=0, writes=i == 0)])
            cache.end_step(plan)
            rows.append(residual)
        outs.append(torch.cat(rows))
    rms = ((outs[0] - outs[1]).pow(2).mean() / outs[1].pow(2).mean()).sqrt().item()
    # rows of integers: 0.9 % of a product, four of them a block, one behind the other; 2^-9 for each of some eleven roundings to bfloat16 a block
    most = 4 * 0.009 + (0.002 * 11 ** 0.5 if dtype == torch.bfloat16 else 0.0)
    assert 0 < rms <= len(blocks) * most, rms
    assert ops.device_status(dev).tolist() == [0, 0, 0, 0]
