"""Engines whose projections are 8-bit integers, against the plain model with every projection's operands quantised."""
import numpy as np
import pytest
import torch

import qwen3_b200 as q
from helpers import make_folder, random_tokens, tiny
from plain import qwen3_plain as plain

pytestmark = pytest.mark.gpu


def quantised(x):
    """Rows as the values that their codes stand for."""
    top = np.abs(x).max(-1, keepdims=True)
    return np.rint(127 * x / np.where(top > 0, top, 1)) * top / 127


def plain_logits(monkeypatch, cfg, weights, tokens):
    head = plain.output_weight(cfg, weights)

    def linear(x, w, rnd=plain.identity):
        x, w = np.asarray(x, dtype=np.float64), np.asarray(w, dtype=np.float64)
        return x @ w.T if w.shape == head.shape and w is head or np.shares_memory(w, head) else quantised(x) @ quantised(w).T
    with monkeypatch.context() as m:
        m.setattr(plain, "linear", linear)
        return plain.forward(cfg, weights, tokens)


def near(got, want, codes_moved):
    """32-bit sums in another order move a value by some units, and one in some ten thousand next to a tie by a whole code, 1/127 of its row's largest.
    So nearly all logits agree to 1e-4 of the largest one, and none is further off than a few moved codes can bring it."""
    got, want = np.asarray(got, dtype=np.float64), np.asarray(want)
    off = np.abs(got - want) / np.abs(want).max()
    assert off.max() <= codes_moved, off.max()
    return off


@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
def test_32_bit_engine(tmp_path, monkeypatch, name):
    cfg = tiny(name)
    folder, weights = make_folder(tmp_path, cfg, seed=3)
    engine = q.Engine.from_folder(folder, dtype="float32", max_tokens=64 * 8, weight_dtype="int8", guard_scratch=True)
    rng = np.random.default_rng(5)
    prompts = [random_tokens(rng, n, cfg["vocab_size"]) for n in (9, 1, 30)]
    slots = [engine.new_sequence() for _ in prompts]
    got = engine.step([q.StepEntry(s, p, want=range(len(p))) for s, p in zip(slots, prompts)]).cpu().numpy()
    offs, at = [], 0
    for p in prompts:
        offs.append(near(got[at:at + len(p)], plain_logits(monkeypatch, cfg, weights, p), 0.03))
        at += len(p)
    for _ in range(3):                                     # single tokens, from a captured graph
        new = random_tokens(rng, len(prompts), cfg["vocab_size"])
        prompts = [p + [t] for p, t in zip(prompts, new)]
        got = engine.step([q.StepEntry(s, [t], want=[0]) for s, t in zip(slots, new)]).cpu().numpy()
        for row, p in zip(got, prompts):
            offs.append(near(row, plain_logits(monkeypatch, cfg, weights, p)[-1], 0.03))
    assert np.median(np.concatenate([o.ravel() for o in offs])) <= 1e-4
    assert engine.scratch_violations() == []
    exact = plain.forward(cfg, weights, prompts[0])
    assert np.abs(plain_logits(monkeypatch, cfg, weights, prompts[0]) - exact).max() > 1e-3 * np.abs(exact).max()      # (the codes are felt)


@pytest.mark.parametrize("name", ["A", "C", "D"])
def test_bfloat16_engine(tmp_path, monkeypatch, name):
    """Beside the plain model with codes and bfloat16's roundings, which move codes: as far as these move the logits, four times over."""
    cfg = tiny(name)
    folder, weights = make_folder(tmp_path, cfg, seed=4)
    engine = q.Engine.from_folder(folder, dtype="bfloat16", max_tokens=64 * 8, weight_dtype="int8", guard_scratch=True)
    tokens = random_tokens(np.random.default_rng(6), 40, cfg["vocab_size"])
    slot = engine.new_sequence()
    got = engine.step([q.StepEntry(slot, tokens, want=range(40))]).cpu().numpy().astype(np.float64)
    exact = plain_logits(monkeypatch, cfg, weights, tokens)
    rounded = plain.forward(cfg, weights, tokens, rnd=plain.round_bf16, rnd_logits=plain.identity)
    unrounded = plain.forward(cfg, weights, tokens)
    bound = 4 * np.abs(rounded - unrounded).max() + 0.03 * np.abs(exact).max()
    assert np.abs(got - exact).max() <= bound
    assert engine.scratch_violations() == []


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_steps_from_graphs_and_launched(dtype):
    """The same kernels, the same bits; and a sequence's tokens do not hang on the slots beside it in a product."""
    config = q.config_from_dict(tiny("B"))
    outs = []
    for graphs in (True, False):
        engine = q.Engine.from_random(config, 7, dtype=dtype, max_tokens=64 * 8, weight_dtype="int8", use_graphs=graphs)
        slots = [engine.new_sequence() for _ in range(3)]
        engine.step([q.StepEntry(s, [5 + s, 6, 7]) for s in slots])
        outs.append(torch.cat([engine.step([q.StepEntry(s, [9 + i], want=[0]) for s in slots]).clone() for i in range(3)]))
        engine.check_kernels()
    assert torch.equal(outs[0], outs[1])


def test_checkpoints_are_quantised_as_they_are_stored(tmp_path):
    """A 32-bit checkpoint is not rounded to bfloat16 before it is quantised, whichever way it comes; what was read for it is given back."""
    cfg = tiny("A", torch_dtype="float32")
    folder, weights = make_folder(tmp_path, cfg, seed=8, storage="float32")
    name = [n for n in weights if n.endswith("down_proj.weight")][0]
    want = quantised(weights[name])
    for dtype in ("bfloat16", "float32"):
        model = q.Engine.from_folder(folder, dtype=dtype, max_tokens=64, weight_dtype="int8").model
        w = model.blocks[0].feed_forward.w_down
        assert w.codes.dtype == torch.int8 and np.abs(w.float().double().cpu().numpy() - want).max() <= 1e-6 * np.abs(want).max()
        memory = q.build_model(q.load_config(folder).plan())
        memory.bind(q.load_weights(folder, memory.weight_specs(), memory.ignorable_names()), torch.bfloat16 if dtype == "bfloat16" else torch.float32,
                    "cuda", eight_bit=True)
        for a, b in zip(model.blocks, memory.blocks):
            for x, y in ((a.mixer.w_qkv, b.mixer.w_qkv), (a.mixer.w_o, b.mixer.w_o), (a.feed_forward.w_gate_up, b.feed_forward.w_gate_up), (a.feed_forward.w_down, b.feed_forward.w_down)):
                assert torch.equal(x.codes, y.codes) and torch.equal(x.scales, y.scales)


def test_memory_of_a_checkpoint_in_8_bits(tmp_path):
    config = q.config_from_dict(tiny("B", num_hidden_layers=6, hidden_size=512, intermediate_size=2048))
    folder = str(tmp_path / "model")
    q.write_random_model(folder, config, 2)
    held = {}
    for weight_dtype in (None, "int8"):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        engine = q.Engine.from_folder(folder, dtype="bfloat16", max_tokens=64, max_seq_len=64, weight_dtype=weight_dtype)
        held[weight_dtype] = torch.cuda.memory_allocated() - before
        del engine
    layer = 2 * (512 * 2048 * 3 + 512 * 10 * 32 + 512 * 256)
    assert held[None] - held["int8"] >= 0.45 * 6 * layer


def test_other_models_are_refused():
    from dozazen_cases import case
    with pytest.raises(ValueError, match="8 bits"):
        q.Engine.from_random(q.config_from_dict(case("A")), 1, max_tokens=64, weight_dtype="int8")


@pytest.mark.parametrize("cache_dtype", [None, "float8"])
def test_with_drafted_tokens(cache_dtype):
    """8-bit weights under either cache: drafted tokens against the same tokens one by one, and generation with drafts."""
    config = q.config_from_dict(dict(tiny("D"), torch_dtype="bfloat16"))
    outs = []
    for tree in (True, False):
        engine = q.Engine.from_random(config, 5, dtype="float32", max_tokens=512, weight_dtype="int8", cache_dtype=cache_dtype)
        slot = engine.new_sequence()
        engine.step([q.StepEntry(slot, list(range(20)))])
        if tree:
            outs.append(engine.step_tree([q.TreeEntry(slot, [3, 4, 5], [-1, 0, 1])]).clone())
            engine.keep({slot: [0, 1, 2]})
        else:
            outs.append(torch.cat([engine.step([q.StepEntry(slot, [t], want=[0])]).clone() for t in (3, 4, 5)]))
    assert float((outs[0] - outs[1]).abs().max()) <= 0.03 * float(outs[0].abs().max())
    engine = q.Engine.from_random(config, 5, dtype="bfloat16", max_tokens=512, weight_dtype="int8", cache_dtype=cache_dtype)
    results = q.generate_speculative(engine, [[5, 6, 7] * 8, [3, 9] * 10], 8)
    assert [len(r.token_ids) for r in results] == [8, 8] and engine.cache.pages_held() == 0
    results = q.generate_token_ids(engine, [[5, 6, 7] * 8, [3, 9] * 10], q.SamplingParams(mode="greedy"), q.GenerationOptions(max_new_tokens=8))
    assert [len(r.token_ids) for r in results] == [8, 8]
