"""Every kind of layer that takes 8-bit weights, against the same layer with the operands of its projections quantised in 64 bits.

The engine beside the 8-bit one runs the 32-bit kernels; its products are replaced by ones that quantise both operands, multiply the values that the codes stand for, and round
once.  Both norm in 32 bits, so a value moves by some units, and a code where that brings it over a tie: one in some ten thousand, by 1/127 of the row's
largest.  So nearly all logits agree to 1e-4 of the largest one, and none is further off than a few such codes can bring it (0.03: the same bounds as
of the engines beside the plain model)."""
import dataclasses

import numpy as np
import pytest
import torch

import qwen3_b200 as q
from helpers import random_tokens, tiny

pytestmark = pytest.mark.gpu
SMALL = dict(hidden_size=96, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=32, intermediate_size=160, vocab_size=301,
             max_position_embeddings=1024)
WIDE = dict(SMALL, hidden_size=768, num_attention_heads=12, num_key_value_heads=4, head_dim=64, intermediate_size=2048, max_position_embeddings=4096)
ROPE = {"head_dim": 32, "theta": 1e4, "max_positions": 1024}


def quantised(x):
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    return torch.where(top > 0, (127 * x / top).round() * top / 127, torch.zeros_like(x))


def product(x, w, out):
    return out.copy_(quantised(x) @ quantised(w).t())


def plan_of(sizes, mixer=None, feed_forward=None, layers=None):
    plan = q.config_from_dict(tiny("A", **sizes)).plan()
    changed = []
    for i, s in enumerate(plan.layers):
        m = dict(s.mixer.params, **(mixer or {}), **(layers[i] if layers else {}))
        f = dict(s.feed_forward.params, **(feed_forward or {}))
        changed.append(dataclasses.replace(s, mixer=q.PartSpec(s.mixer.kind, m), feed_forward=q.PartSpec(s.feed_forward.kind, f)))
    return dataclasses.replace(plan, layers=changed)


def engines(plan, config, dtype, seed=5, **kwargs):
    """The 8-bit engine, and the one whose products quantise their operands (None for that of another type)."""
    from qwen3_b200.engine.engine import Engine
    specs = q.build_model(plan).weight_specs()
    tensors = q.random_weights(specs, seed, dtype=torch.float32, device="cuda")
    for name, t in tensors.items():                        # (drawn around zero, where biases and sinks would not be felt)
        if specs[name].role == "bias":
            tensors[name] = t * 20
    out = []
    for eight_bit in (True, False):
        model = q.build_model(plan)
        model.bind(dict(tensors), dtype, "cuda", eight_bit)
        out.append(Engine(model, config, max_tokens=4096, max_seq_len=min(plan.max_positions, 2048), use_graphs=eight_bit, **kwargs))
    return out


def run(engine, prompts, news, patched, monkeypatch):
    """Logits of all prompts at once, then of single tokens."""
    from qwen3_b200.parts import attention, mlp
    with monkeypatch.context() as m:
        if patched:
            m.setattr(attention, "linear", product)
            m.setattr(mlp, "linear", product)
        slots = [engine.new_sequence() for _ in prompts]
        outs = [engine.step([q.StepEntry(s, p, want=range(max(0, len(p) - 40), len(p))) for s, p in zip(slots, prompts)]).double().cpu().numpy().copy()]
        for new in news:
            outs.append(engine.step([q.StepEntry(s, [t], want=[0]) for s, t in zip(slots, new)]).double().cpu().numpy().copy())
        engine.check_kernels()
    return np.concatenate(outs)


def compare(plan, sizes, monkeypatch, lengths=(70, 1, 9), median=1e-4):
    config = q.config_from_dict(tiny("A", **sizes))
    assert q.build_model(plan).takes_eight_bit()
    rng = np.random.default_rng(7)
    prompts = [random_tokens(rng, n, sizes["vocab_size"]) for n in lengths]
    news = [random_tokens(rng, len(lengths), sizes["vocab_size"]) for _ in range(4)]
    got, want = (run(e, prompts, news, patched, monkeypatch) for e, patched in zip(engines(plan, config, torch.float32, guard_scratch=True), (False, True)))
    off = np.abs(got - want) / np.abs(want).max()
    assert np.isfinite(got).all() and off.max() <= 0.03 and np.median(off) <= median, (off.max(), np.median(off))


OPTIONS = [{}, {"position": None}, {"qk_norm": None}, {"out_bias": True}, {"bias": True}, {"bias": True, "out_bias": True, "qk_norm": None}, {"window": 32},
           {"chunk": 32}, {"value_dim": 48}, {"softcap": 5.0}, {"sink": True}, {"learned_sink": True}, {"value_heads": 1}, {"out_float32": True},
           {"window": 32, "keep_first": 2}, {"conv_taps": 4}, {"conv_taps": 1}, {"window": 64, "pool": 16}, {"tied_values": True},
           {"value_position": q.PartSpec("rope", ROPE)}, {"out_gate": True}, {"out_gate": True, "window": 32}, {"norm_once": True},
           {"norm_once": True, "temperature": {"coef": 0.1, "every": 8}}, {"distance_bias": 64, "bias_rows": 32},
           {"qk_norm": None, "position": q.PartSpec("rope", dict(ROPE, interleaved=True))},
           {"qk_norm": None, "bias": True, "conv_taps": 3, "position": q.PartSpec("rope", dict(ROPE, interleaved=True))}]


@pytest.mark.parametrize("options", OPTIONS, ids=lambda o: "-".join(o) or "plain")
def test_attention(monkeypatch, options):
    compare(plan_of(SMALL, mixer=options), SMALL, monkeypatch)


def test_values_that_later_layers_blend_with_the_first_ones(monkeypatch):
    compare(plan_of(SMALL, layers=[{"value_mix": "first", "bias": True}, {"value_mix": "blend", "bias": True}]), SMALL, monkeypatch)


def test_a_layer_on_another_layers_cache(monkeypatch):
    plan = plan_of(dict(SMALL, num_hidden_layers=3), layers=[{}, {}, {"shared_kv": True}])
    plan = dataclasses.replace(plan, layers=plan.layers[:2] + [dataclasses.replace(plan.layers[2], cache_from=0)])
    compare(plan, SMALL, monkeypatch)


@pytest.mark.parametrize("options", [{"activation": "gelu_tanh"}, {"activation": "clamped", "limit": 0.5}, {"intermediate_size": 60},
                                     {"intermediate_size": 60, "activation": "gelu_tanh"}, {"intermediate_size": 60, "activation": "clamped"}],
                         ids=lambda o: "-".join(map(str, o.values())))
def test_feed_forward(monkeypatch, options):
    compare(plan_of(SMALL, feed_forward=options), SMALL, monkeypatch)


@pytest.mark.parametrize("options", [{}, {"out_gate": True, "bias": True}])
def test_prompts_of_every_form_of_the_products(monkeypatch, options):
    """Steps of a few, some hundred and more than a thousand tokens.

    The median is another one here.  A token of this model has 2 (3 * 768 + 2,048) = 8,700 codes, where that of the small one has 900, and reads those of up to 1,500
    others: with one code moved in some ten thousand nearly every token has one.  One code of a row of K values, whose largest is c times their root mean square (c some
    3.3), moves the row by c / (127 sqrt(K)) = 0.0009 of its norm, so the next row's ratios by 127 / c times that, 0.036 of a code, so that one code in 28 moves there: c /
    127 sqrt(1 / 28) = 0.005 of the norm; and so on towards c / 127 / sqrt(6) = 0.011, where the two engines' roundings have nothing in common (each is off by
    c / 127 / sqrt(12)).  Eight such products in a row, added up in squares: 0.03 of a logit's root mean square, which is a quarter of the largest one; half of all
    values of a normal distribution are below 0.67 of that: 0.005."""
    from qwen3_b200.csrc import ops
    forms, plain = set(), ops.int8_plan
    monkeypatch.setattr(ops, "int8_plan", lambda M, N, K: forms.add(plain(M, N, K)[0]) or plain(M, N, K))
    plan = plan_of(WIDE, mixer=options)
    for lengths in ((3, 1), (40, 60), (300, 7), (1500, 800)):
        compare(plan, WIDE, monkeypatch, lengths, median=0.005)
    assert forms == {"few", "mid", "pair"}


@pytest.mark.parametrize("sizes,lengths", [(SMALL, (70, 1, 9)), (WIDE, (300, 7)), (WIDE, (1500, 800))])
@pytest.mark.parametrize("options", [{}, {"bias": True, "sink": True}, {"out_gate": True}, {"out_float32": True}, {"conv_taps": 4}])
def test_bfloat16(monkeypatch, sizes, lengths, options):
    """Beside the 32-bit engine on the same codes: as far as bfloat16's roundings move the logits of the unquantised engines, four times over, and a few moved codes."""
    plain_options = {} if options.get("out_float32") else options          # (products of 16-bit engines take no 32-bit rows)
    config = q.config_from_dict(tiny("A", **sizes))
    rng = np.random.default_rng(8)
    prompts = [random_tokens(rng, n, sizes["vocab_size"]) for n in lengths]
    news = [random_tokens(rng, len(lengths), sizes["vocab_size"]) for _ in range(3)]
    logits = {}
    for dtype in (torch.float32, torch.bfloat16):
        logits[dtype, True] = run(engines(plan_of(sizes, mixer=options), config, dtype)[0], prompts, news, False, monkeypatch)
        logits[dtype, False] = run(engines(plan_of(sizes, mixer=plain_options), config, dtype)[1], prompts, news, False, monkeypatch)
    exact = logits[torch.float32, True]
    moved = np.abs(logits[torch.bfloat16, False] - logits[torch.float32, False]).max()
    assert np.abs(logits[torch.bfloat16, True] - exact).max() <= 4 * moved + 0.03 * np.abs(exact).max()
