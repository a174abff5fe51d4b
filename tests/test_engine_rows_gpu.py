"""Engines over a cache in 8 bits and with drafted tokens: models that do not take them, and what a step may not leave behind."""
import pytest
import torch

import qwen3_b200 as q
from helpers import tiny
from test_takes_rows import plan_with, shifted_plan

pytestmark = pytest.mark.gpu


class Config:
    """A configuration that is only a plan."""
    torch_dtype = "float32"

    def __init__(self, plan):
        self._plan = plan

    def plan(self):
        return self._plan


@pytest.mark.parametrize("taps", [1, 4])
def test_a_convolution_over_the_rows_is_refused(taps):
    config = Config(plan_with(conv_taps=taps))
    with pytest.raises(ValueError):
        q.Engine.from_random(config, 1, dtype="float32", max_tokens=256, cache_dtype="float8")
    engine = q.Engine.from_random(config, 1, dtype="float32", max_tokens=256)
    slot = engine.new_sequence()
    engine.step([q.StepEntry(slot, [1, 2, 3], want=[2])])
    with pytest.raises(q.StepError):
        engine.step_tree([q.TreeEntry(slot, [1], [-1])])
    assert engine.length(slot) == 3


@pytest.mark.parametrize("cache_dtype", [None, "float8"])
def test_blocks_that_keep_a_row_are_refused_drafted_tokens(cache_dtype):
    """Their steps go over either cache: a sequence run whole is the sequence run in pieces and token by token."""
    engine = q.Engine.from_random(Config(shifted_plan()), 2, dtype="float32", max_tokens=512, cache_dtype=cache_dtype)
    tokens = [(7 * i) % 251 for i in range(80)]
    outs = []
    for cuts in ([80], [40, 30, 10], [76, 1, 1, 1, 1]):
        slot, at = engine.new_sequence(), 0
        for n in cuts:
            last = engine.step([q.StepEntry(slot, tokens[at:at + n], want=[n - 1])])
            at += n
        outs.append(last.clone())
        with pytest.raises(q.StepError):
            engine.step_tree([q.TreeEntry(slot, [1, 2, 3], [-1, 0, 0])])
        assert engine.length(slot) == 80
        engine.release(slot)
    # 32-bit sums in another order, and over 8 bits one rounding of a row that they turn
    bound = (2e-4 if cache_dtype is None else 0.02) * float(outs[0].abs().max())
    assert all(float((o - outs[0]).abs().max()) <= bound for o in outs)


def test_a_kernel_that_gave_up_ends_the_generation():
    """The word that a kernel sets when a wait runs out is set by hand, between steps: the tokens of that step are not returned, the slots and
    pages go back, and the next generation runs."""
    from qwen3_b200.csrc import ops
    engine = q.Engine.from_random(Config(plan_with()), 3, dtype="float32", max_tokens=512)
    calls = [0]

    def draft(text):
        calls[0] += 1
        if calls[0] == 3:
            ops._status_word(engine.device).fill_(47)
        return [1, 2], [-1, 0]
    with pytest.raises(ops.KernelError, match="47.*drafted"):
        q.generate_speculative(engine, [[5, 6, 7]], 20, draft=draft)
    assert engine.cache.pages_held() == 0 and calls[0] == 3
    assert len(q.generate_speculative(engine, [[5, 6, 7]], 5, draft=draft)[0].token_ids) == 5


def test_the_status_word_is_the_devices_however_it_is_named():
    """Kernels write into the word of the device that their tensors name ("cuda:0"); an engine or a caller may have named it "cuda"."""
    from qwen3_b200.csrc import ops
    engine = q.Engine.from_random(Config(plan_with()), 3, dtype="float32", max_tokens=512, device="cuda")
    engine.check_kernels()
    for name in ("cuda", torch.device("cuda"), torch.device("cuda", torch.cuda.current_device())):
        ops._status_word(torch.zeros(1, device="cuda").device).fill_(48)
        assert ops.tcgen05_status(name) == 48 and ops.tcgen05_status(name) == 0
    ops._status_word(torch.zeros(1, device="cuda").device).fill_(48)
    with pytest.raises(ops.KernelError):
        engine.check_kernels()


@pytest.mark.parametrize("name,dtype", [("D", "bfloat16"), ("C", "bfloat16"), ("A", "float32")])
def test_a_step_reads_back_the_pages_that_it_holds(monkeypatch, name, dtype):
    """One prompt beside single tokens of sequences of very unequal length: the buffers hold the sequences' pages, not as many for each as the
    longest has, and every token has the logits that it has where the prompt runs by itself and the others attend to the pages as they are."""
    from qwen3_b200.parts import attention
    monkeypatch.setattr(attention, "rows_at_once", 64)
    config = q.config_from_dict(dict(tiny(name, max_position_embeddings=512), torch_dtype="bfloat16"))
    lengths, outs = [400] + [5 + i for i in range(12)] + [64], []
    prompt = [(5 * i) % 200 for i in range(90)]
    for together in (True, False):
        engine = q.Engine.from_random(config, 5, dtype=dtype, max_tokens=64 * 40, cache_dtype="float8", guard_scratch=True)
        slots = [engine.new_sequence() for _ in lengths]
        for s, n in zip(slots, lengths):                                  # (one by one: what is read back by then is small)
            for at in range(0, n, 64):
                engine.step([q.StepEntry(s, [(3 * i + s) % 200 for i in range(at, min(at + 64, n))])])
        engine.scratch = type(engine.scratch)(engine.device, guard=True)
        new = engine.new_sequence()
        ones, run = [q.StepEntry(s, [9], want=[0]) for s in slots], [q.StepEntry(new, prompt, want=[0, 50, 89])]
        outs.append(engine.step(ones + run).clone() if together else torch.cat([engine.step(ones).clone(), engine.step(run).clone()]))
        assert engine.scratch_violations() == []
        read = [t.numel() for k, t in engine.scratch._flat.items() if k[0] == "attn.read_keys"]
        pages = (sum(-(-(n + 1) // 64) for n in lengths) if together else 0) + 2
        assert read == [pages * 64 * config.num_key_value_heads * config.head_dim]
    # as the bound of the two ways over one sequence: a rounding of a layer's rows to the compute type, which can move a code by one of its steps
    bound = 0.06 if dtype == "bfloat16" else 0.02
    assert float((outs[0] - outs[1]).abs().max()) <= bound * float(outs[0].abs().max())


@pytest.mark.parametrize("cache_dtype,sequences,positions,want", [(None, 80, 2048, "mma"), ("float8", 40, 8192, "tc"), (None, 40, 2048, "tc"), ("float8", 80, 8192, "mma")])
def test_the_form_goes_by_the_steps_lengths(monkeypatch, cache_dtype, sequences, positions, want):
    """Page tables of an engine are as wide as its longest sequence may become; which kernel takes a step of 20 rows a kv head goes by what the
    sequences hold: 160 items of a page each are many for tcgen05 over bfloat16, 80 are not over 8 bits."""
    from qwen3_b200.csrc import ops
    config = q.config_from_dict(dict(tiny("D", max_position_embeddings=positions), torch_dtype="bfloat16"))
    engine = q.Engine.from_random(config, 5, dtype="bfloat16", max_tokens=64 * max(sequences, positions // 64), n_slots=sequences, cache_dtype=cache_dtype)
    assert engine.cache.pages_per_slot == positions // 64
    slots, names, call = [engine.new_sequence() for _ in range(sequences)], [], ops._call_packed

    def recorded(what, source, name, *a):
        names.append(name)
        return call(what, source, name, *a)
    monkeypatch.setattr(ops, "_call_packed", recorded)
    engine.step([q.StepEntry(s, [1 + s % 50, 2]) for s in slots])
    names.clear()
    engine.step_tree([q.TreeEntry(s, [3] * 10, list(range(-1, 9))) for s in slots])
    engine.keep({s: [] for s in slots})
    assert [n for n in names if "tree" in n] == [f"q3_attention_tree_{want}_bf16"] * 2
