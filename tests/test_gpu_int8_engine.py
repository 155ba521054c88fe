"""The engine with its layers' matrices as 8-bit integers, against a plain model in 64 bits that rounds where the engine does.

Both round the same numbers to integers, but not from the same bits, and a rounding to integers does not let small differences stay small.  A row's step is
s = max|x| / 127, with the largest entry some 4 times the row's root mean square 0.03 of that.  Entries that differ by d (of the root mean square) lie on two sides
of a border in d / s of the cases, each then by s: what comes out differs by sqrt(d / s) s = sqrt(d s).  float32's 1e-6 so becomes 2e-4 behind the first product,
2e-3, 8e-3 and 1.5e-2 behind the next three, and tends to s itself, which is where bfloat16 (2^-9 is a quarter of the largest entries' step) begins.  As far as that
goes both are bounded by integers that differ by one everywhere: s / sqrt(12) = 0.9 % a product, 3 % over the twelve of three layers in quadrature.  bfloat16 has the 1.5 %
beside it that the engine has without integers: 5 %.  The largest of all logits' errors is allowed four times the root mean square's share.  (What each
operator does exactly is tested for itself; here it is whether they stand in the right places.)"""
from dataclasses import replace

import numpy as np
import pytest
import torch

import helpers
from plain.hunyuan_plain import PlainModel, causal_attention, neox_rope, rms_norm, swiglu

RMS = {"float32": 3e-2, "bfloat16": 5e-2}


def _rounded(x):
    """What the 8-bit rows of x stand for."""
    top = x.abs().amax(-1, keepdim=True)
    return torch.nan_to_num(torch.round(127 * x / top)) * top / 127


class RoundedModel(PlainModel):
    """The plain model with every product of a layer taken of rounded rows and rounded weights."""

    def __init__(self, folder):
        super().__init__(folder, torch.float64)
        self.r = {n: _rounded(w) for n, w in self.w.items() if w.dim() == 2 and ".layers." in n}

    def layer(self, h, l, positions):
        c, w, r, p, T = self.cfg, self.w, self.r, f"model.layers.{l}.", h.shape[0]
        n = _rounded(rms_norm(h, w[p + "input_layernorm.weight"], c.eps))
        q, k, v = ((n @ r[p + f"self_attn.{m}_proj.weight"].T).reshape(T, -1, c.head_dim) for m in "qkv")
        q, k = (neox_rope(t, positions, c.rope_dim, self.inv_freq) for t in (q, k))
        if c.qk_norm:
            q = rms_norm(q, w[p + "self_attn.query_layernorm.weight"], c.eps)
            k = rms_norm(k, w[p + "self_attn.key_layernorm.weight"], c.eps)
        h = h + _rounded(causal_attention(q, k, v, c.window)) @ r[p + "self_attn.o_proj.weight"].T
        n = _rounded(rms_norm(h, w[p + "post_attention_layernorm.weight"], c.eps))
        act = swiglu(n @ r[p + "mlp.gate_proj.weight"].T, n @ r[p + "mlp.up_proj.weight"].T)
        return h + _rounded(act) @ r[p + "mlp.down_proj.weight"].T


@pytest.fixture(scope="module")
def rounded_models(model_dirs):
    made = {}
    return lambda name: made.setdefault(name, RoundedModel(model_dirs(name)))


def _close(got, ref, dtype, what):
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    assert got.shape == ref.shape and np.isfinite(got).all(), what
    rms = np.sqrt(((got - ref) ** 2).mean()) / np.sqrt((ref ** 2).mean())
    worst = np.abs(got - ref).max() / np.abs(ref).max()
    assert rms <= RMS[dtype] and worst <= 4 * RMS[dtype], f"{what}: rms {rms:.2e}, worst {worst:.2e}"


def _engine(folder, dtype, **kw):
    from hymt2sharp_b200 import Engine
    return Engine(folder, dtype=dtype, weights="int8", **{"max_tokens": 2048, **kw})


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "W", "M", "H", "HW", "S"])
def test_prompts_and_steps_of_unequal_sequences(name, dtype, model_dirs, rounded_models):
    from hymt2sharp_b200 import StepEntry
    plain = rounded_models(name)
    eng = _engine(model_dirs(name), dtype, max_batch=3)
    for s in eng.cache.storage:
        s.fill_(float("nan"))
    lens = (150, 3, 65)
    seqs = [helpers.random_tokens(plain.cfg.vocab, n + 6, 70 + i) for i, n in enumerate(lens)]
    slots = eng.alloc_slots(3)
    out = eng.step([StepEntry(s, q[:n], list(range(n))) for s, q, n in zip(slots, seqs, lens)]).cpu().numpy()
    got = [list(out[sum(lens[:i]):sum(lens[:i + 1])]) for i in range(3)]
    for step in range(4):
        for row, i in zip(eng.step([StepEntry(slots[i], [seqs[i][lens[i] + step]], [0]) for i in range(3)]).cpu().numpy(), range(3)):
            got[i].append(row)
    for row in eng.step([StepEntry(slots[2], seqs[2][lens[2] + 4:], [0, 1])]).cpu().numpy():
        got[2].append(row)
    eng.check()
    for i, n in enumerate(lens):
        _close(np.stack(got[i]), plain.logits(seqs[i][:n + (6 if i == 2 else 4)]).numpy(), dtype, f"{name} {dtype} sequence {i}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["B", "H"])
def test_generation_through_graphs_is_generation_step_by_step(name, dtype, model_dirs):
    from hymt2sharp_b200 import StepEntry
    eng = _engine(model_dirs(name), dtype, max_batch=3)
    prompts = [helpers.random_tokens(eng.vocab, n, 5 + n) for n in (70, 2, 9)]
    out = eng.generate(prompts, max_new_tokens=12)
    slots = eng.alloc_slots(3)
    logits = eng.step([StepEntry(s, q, [len(q) - 1]) for s, q in zip(slots, prompts)])
    tokens = [[int(t)] for t in logits.argmax(1)]
    for _ in range(11):
        logits = eng.step([StepEntry(s, [t[-1]], [0]) for s, t in zip(slots, tokens)])
        for t, n in zip(tokens, logits.argmax(1)):
            t.append(int(n))
    eng.check()
    assert [r.tokens for r in out.results] == tokens


@pytest.mark.gpu
@pytest.mark.parametrize("name, one_call", [("M", True), ("H", True), ("HW", True), ("B", False)])
def test_a_prompts_block_by_one_call_is_its_parts_one_by_one(name, one_call, model_dirs, monkeypatch):
    """Heads of 64 and 128, with and without a window, prompts and a further piece of one: logits and the number of launches."""
    from hymt2sharp_b200 import StepEntry
    from hymt2sharp_b200.kernels import ops
    eng = _engine(model_dirs(name), "bfloat16", max_batch=2)
    calls, launch = [], ops.dense_block_q8
    monkeypatch.setattr(ops, "dense_block_q8", lambda *args: (calls.append(1), launch(*args)))
    seqs = [helpers.random_tokens(eng.vocab, n, n) for n in (203, 31)]
    results = []
    for whole in (True, False):
        for block in eng.model.blocks:
            block.dense_rows8 = block.dense_rows8 and whole
        slots, before, logits = eng.alloc_slots(2), ops.launches, []
        for cut in (slice(0, 20), slice(20, 203)):
            entries = [StepEntry(s, q[cut], list(range(len(q[cut])))) for s, q in zip(slots, seqs)]
            logits.append(eng.step(entries).clone())
        results.append((torch.cat(logits), ops.launches - before, len(calls)))
        eng.free_slots(slots)
    eng.check()
    (a, na, ca), (b, nb, cb) = results
    assert torch.equal(a, b) and na == nb and ca == (2 * len(eng.model.blocks) if one_call else 0) and cb == ca


@pytest.mark.gpu
def test_the_layers_matrices_are_held_once_and_in_8_bits(model_dirs):
    from hymt2sharp_b200 import Engine
    stored, small = Engine(model_dirs("H"), dtype="bfloat16", max_tokens=256), _engine(model_dirs("H"), "bfloat16", max_tokens=256)
    a, b = stored.model, small.model
    layers = sum(p.numel() for blk in a.blocks for p in (blk.mixer.qkv.weight, blk.mixer.out.weight, blk.feed_forward.gate_up.weight, blk.feed_forward.down.weight))
    scales = sum(4 * p.shape[0] for blk in a.blocks for p in (blk.mixer.qkv.weight, blk.mixer.out.weight, blk.feed_forward.gate_up.weight, blk.feed_forward.down.weight))
    assert a.streamed_weight_bytes() - b.streamed_weight_bytes() == layers - scales
    blk = b.blocks[0]
    assert blk.mixer.qkv.weight.dtype == torch.int8 and blk.mixer.out_store.weight is blk.mixer.out.weight and blk.feed_forward.down_store.weight is blk.feed_forward.down.weight
    # what they stand for is within half a step of what is stored
    w = a.blocks[0].mixer.qkv.weight.float()
    v = blk.mixer.qkv.rows.values(torch.float32)
    assert ((v - w).abs() <= w.abs().amax(1, keepdim=True) / 254 * (1 + 1e-5)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("general", [dict(value_dim=24), dict(norm_first=True), dict(sink=True), dict(head_gate="gate.weight")])
def test_attention_in_its_general_forms_takes_8_bit_rows(general, tmp_path):
    """The projections of the forms beyond the classic one, and a clamped gated feed-forward, in a pre-norm block: against the same block with the
    matrices that the integers stand for, as far as the rounding of the rows may move it (0.9 % a product, four of them one behind the other)."""
    from hymt2sharp_b200.cache import PagedCache
    from hymt2sharp_b200.engine.engine import StepEntry, make_context
    from hymt2sharp_b200.kernels import ops
    from hymt2sharp_b200.parts.base import MixerSlot, PartSpec, build_part
    dev, hidden, heads, d = "cuda:0", 96, 4, 32
    attn = dict(hidden=hidden, heads=heads, kv_heads=2, head_dim=d, eps=1e-5, qk_norm=True, position=None, q_proj="q", k_proj="k", v_proj="v", o_proj="o",
                q_norm="qn", k_norm="kn", **general)
    ff = dict(hidden=hidden, intermediate=200, limit=2.0, alpha=1.702, gate_proj="g", up_proj="u", down_proj="d", gate_bias="gb", up_bias="ub", down_bias="db")
    norm = lambda n: PartSpec("rmsnorm", dict(dim=hidden, eps=1e-5, weight=n))
    torch.manual_seed(3)
    made = lambda weights: build_part("block", PartSpec("pre_norm", dict(norm1=norm("n1"), mixer=PartSpec("gqa_attention", {**attn, "weights": weights}),
                                                                      norm2=norm("n2"), feed_forward=PartSpec("clamped_glu", {**ff, "weights": weights}))))
    block8, block = made("int8"), made(None)
    stored = {n: torch.randn(s.shape) * (1 / s.shape[-1] ** 0.5 if len(s.shape) == 2 else 0.1) + (1.0 if s.init == "gain" else 0.0)
              for n, s in block.tensors().items()}
    same = {n: _rounded(w.double()).float() if w.dim() == 2 else w for n, w in stored.items()}
    outs = []
    for b, weights in ((block8, stored), (block, same)):
        b.load(weights, torch.device(dev), torch.float32)
        need = replace(b.cache_needs()[0], planes=1)
        cache = PagedCache([need], torch.float32, torch.device(dev), capacity_tokens=256, block_tokens=64, max_slots=2, state_bytes=0)
        slots = cache.alloc_slots(2)
        ctx, _, _, plan = make_context(cache, [StepEntry(s, [0] * n) for s, n in zip(slots, (40, 7))], 10, torch.float32, dev, ops.device_status(torch.device(dev)))
        torch.manual_seed(4)
        residual = torch.randn(47, hidden, device=dev)
        b.forward(residual, ctx, [MixerSlot(group=0, plane=0)])
        cache.end_step(plan)
        outs.append(residual)
    rms = ((outs[0] - outs[1]).pow(2).mean() / outs[1].pow(2).mean()).sqrt().item()
    assert 0 < rms <= 4 * 0.009, rms
    assert ops.device_status(torch.device(dev)).tolist() == [0, 0, 0, 0]


def test_other_weights_and_other_layers_are_refused(tmp_path):
    import gomerax_models
    import pemezen_models
    from hymt2sharp_b200.config import HunyuanDenseConfig
    from hymt2sharp_b200.engine.engine import Engine, EngineError
    from hymt2sharp_b200.engine.hunyuan_dense import build_spec
    from hymt2sharp_b200.engine.spec import with_weights
    from hymt2sharp_b200.config.registry import get_architecture
    with pytest.raises(EngineError, match="weights must be one of"):
        Engine(str(tmp_path), weights="int4")
    spec = build_spec(HunyuanDenseConfig.from_dict(helpers.CONFIGS["A"]["config"]))
    assert with_weights(spec, None) is spec
    with pytest.raises(ValueError, match="not known"):
        with_weights(spec, "int4")
    small = with_weights(spec, "int8")
    assert small.weights == "int8" and all(l.params[n].params["weights"] == "int8" for l in small.layers for n in ("mixer", "feed_forward"))
    assert spec.weights is None and not any("weights" in l.params[n].params for l in spec.layers for n in ("mixer", "feed_forward"))     # (the caller's is left alone)
    for models, name in ((pemezen_models, "Pemezen"), (gomerax_models, "Gomerax")):
        arch = get_architecture(name)
        other = arch.build_spec(arch.config_class.from_dict(models.CONFIGS["even"]["config"]))
        with pytest.raises(ValueError, match="are built for pre_norm blocks"):
            with_weights(other, "int8")
