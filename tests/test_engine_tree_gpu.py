"""The engine over a cache in 8 bits, and its steps with drafted tokens."""
import numpy as np
import pytest
import torch

from helpers import make_folder, random_tokens, tiny

pytestmark = pytest.mark.gpu


def engine_of(tmp_path, name, dtype, cache_dtype=None, seed=3, **kw):
    import qwen3_b200 as q
    folder, _ = make_folder(tmp_path, tiny(name), seed, name=f"{name}{dtype}")
    kw.setdefault("max_tokens", 1024)
    return q.Engine.from_folder(folder, dtype=dtype, cache_dtype=cache_dtype, **kw)


def run_chain(engine, tokens):
    """Logits of every token of a sequence, its prompt in one step and the rest one by one."""
    import qwen3_b200 as q
    slot, cut = engine.new_sequence(), max(1, len(tokens) - 5)
    out = [engine.step([q.StepEntry(slot, tokens[:cut], want=list(range(cut)))]).clone()]
    for t in tokens[cut:]:
        out.append(engine.step([q.StepEntry(slot, [t], want=[0])]).clone())
    engine.release(slot)
    return torch.cat(out)


@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("cache_dtype", [None, "float8"])
def test_a_tree_is_its_chains(tmp_path, name, dtype, cache_dtype):
    """Every token of a tree has the logits that it has at the end of its own chain, run token by token; after `keep` the sequence goes on as
    if it had been fed the kept chain alone."""
    import qwen3_b200 as q
    engine = engine_of(tmp_path, name, dtype, cache_dtype)
    rng = np.random.default_rng(5)
    vocab = engine.vocab_size
    prompts = [random_tokens(rng, n, vocab) for n in (9, 70, 1)]
    trees = [([-1, 0, 0, 1, 2, 2, 5], [0, 2, 5, 6]), ([-1], [0]), ([-1, -1, 1, 2, 0], [1, 2, 3])]
    slots = [engine.new_sequence() for _ in prompts]
    engine.step([q.StepEntry(s, p) for s, p in zip(slots, prompts)])
    entries = [q.TreeEntry(s, random_tokens(rng, len(t[0]), vocab), t[0]) for s, t in zip(slots, trees)]
    logits = engine.step_tree(entries).clone()
    # one rounding of a row to 8 bits, or of a logit's terms to the compute type, is what a different order of sums can turn
    tol = 2e-4 if dtype == "float32" and cache_dtype is None else None
    at, chains = 0, []
    for p, e in zip(prompts, entries):
        for i in range(len(e.tokens)):
            chain, n = [], i
            while n >= 0:
                chain.append(e.tokens[n])
                n = e.parents[n]
            chains.append((at, p + chain[::-1]))
            at += 1
    engine.keep({s: t[1] for s, t in zip(slots, trees)})
    assert [engine.length(s) for s in slots] == [len(p) + len(t[1]) for p, t in zip(prompts, trees)]
    goes_on = [random_tokens(rng, 1, vocab) for _ in slots]
    after = engine.step([q.StepEntry(s, t, want=[0]) for s, t in zip(slots, goes_on)]).clone()
    for s in slots:
        engine.release(s)
    scale = float(logits.abs().max())
    bound = tol if tol is not None else (0.02 if dtype == "float32" else 0.06) * scale
    for row, chain in chains:
        want = run_chain(engine, chain)[-1]
        assert float((logits[row] - want).abs().max()) <= bound, (row, float((logits[row] - want).abs().max()), scale)
    for i, (p, e, t) in enumerate(zip(prompts, entries, trees)):
        want = run_chain(engine, p + [e.tokens[n] for n in t[1]] + goes_on[i])[-1]
        assert float((after[i] - want).abs().max()) <= bound
    assert engine.cache.pages_held() == 0


@pytest.mark.parametrize("name,dtype", [("A", "float32"), ("D", "bfloat16"), ("C", "bfloat16")])
def test_a_cache_in_8_bits_is_near_the_other(tmp_path, name, dtype):
    """Prompts (whole, and long enough to be read back), decode steps (captured) and follow-ups: the logits move by what rounding keys and
    values to four bits of mantissa moves them."""
    import qwen3_b200 as q
    engines = [engine_of(tmp_path, name, dtype, c, seed=8) for c in (None, "float8")]
    assert engines[1].cache.bytes_per_token() < (0.55 if dtype == "bfloat16" else 0.3) * engines[0].cache.bytes_per_token()
    rng = np.random.default_rng(1)
    prompts = [random_tokens(rng, n, engines[0].vocab_size) for n in (5, 90, 64)]
    outs = []
    for engine in engines:
        slots = [engine.new_sequence() for _ in prompts]
        got = [engine.step([q.StepEntry(s, p, want=[len(p) - 1]) for s, p in zip(slots, prompts)]).clone()]
        for k in range(3):
            got.append(engine.step([q.StepEntry(s, [7 + k], want=[0]) for s in slots]).clone())
        got.append(engine.step([q.StepEntry(s, p[:3 + 20 * i], want=[0, 1]) for i, (s, p) in enumerate(zip(slots, prompts))]).clone())
        outs.append(torch.cat(got))
        for s in slots:
            engine.release(s)
    off = (outs[0] - outs[1]).abs().mean() / outs[0].abs().mean()
    assert 0 < float(off) < 0.1, float(off)


@pytest.mark.parametrize("name", ["C", "D"])
def test_a_prompt_attends_to_pages_read_back_as_to_the_pages(tmp_path, monkeypatch, name):
    """The same codes and scales, read by the tree's attention or read back for the prompt kernels: only roundings of the compute type differ."""
    import qwen3_b200 as q
    from qwen3_b200.parts import attention
    engine = engine_of(tmp_path, name, "bfloat16", "float8", seed=4)
    prompt = random_tokens(np.random.default_rng(3), 150, engine.vocab_size)
    outs = []
    for limit in (512, 64):
        monkeypatch.setattr(attention, "rows_at_once", limit)
        slot = engine.new_sequence()
        engine.step([q.StepEntry(slot, prompt[:70])])
        outs.append(engine.step([q.StepEntry(slot, prompt[70:], want=[0, 40, 79])]).clone())
        engine.release(slot)
    # a layer's keys and values move by roundings of 2^-9, and those can move a code by one of its steps of 2^-4 at most
    assert float((outs[0] - outs[1]).abs().max()) <= 0.06 * float(outs[0].abs().max())


@pytest.mark.parametrize("cache_dtype", [None, "float8"])
def test_speculative_generation_is_greedy_generation(tmp_path, cache_dtype):
    import qwen3_b200 as q
    engine = engine_of(tmp_path, "A", "float32", cache_dtype)
    rng = np.random.default_rng(2)
    base = random_tokens(rng, 6, engine.vocab_size)
    prompts = [base * 4, random_tokens(rng, 11, engine.vocab_size), base[:2] * 9, [3]]
    want = q.generate_token_ids(engine, prompts, q.SamplingParams(mode="greedy"), q.GenerationOptions(max_new_tokens=40, stop_token_ids=[17]))
    calls = [0]
    step_tree = engine.step_tree

    def counted(entries):
        calls[0] += 1
        return step_tree(entries)
    engine.step_tree = counted
    got = q.generate_speculative(engine, prompts, 40, [17])
    assert [(r.token_ids, r.stop_reason) for r in got] == [(r.token_ids, r.stop_reason) for r in want]
    assert calls[0] < 39                                                 # some drafts stood
    assert [r.token_ids for r in q.generate_speculative(engine, prompts, 40, [17], batch_size=2)] == [r.token_ids for r in want]
    assert [r.token_ids for r in q.generate_speculative(engine, prompts, 40, [17], draft=lambda text: ([], []))] == [r.token_ids for r in want]
    assert engine.cache.pages_held() == 0


def test_speculation_where_pages_are_few(tmp_path):
    import qwen3_b200 as q
    engine = engine_of(tmp_path, "A", "float32", max_tokens=128, max_seq_len=64)
    prompts = [[1, 2, 3] * 14, [5, 6] * 20]
    want = q.generate_token_ids(engine, prompts, q.SamplingParams(mode="greedy"), q.GenerationOptions(max_new_tokens=20))
    got = q.generate_speculative(engine, prompts, 20, draft=q.PromptLookup(tokens=40, depth=20))
    assert [r.token_ids for r in got] == [r.token_ids for r in want] and engine.cache.pages_held() == 0


def test_steps_with_drafts_and_their_refusals(tmp_path):
    import qwen3_b200 as q
    engine = engine_of(tmp_path, "A", "float32", "float8")
    slot, other = engine.new_sequence(), engine.new_sequence()
    engine.step([q.StepEntry(slot, [1, 2]), q.StepEntry(other, [3])])
    for bad in ([], [q.TreeEntry(slot, [], [])], [q.TreeEntry(slot, [1], [])], [q.TreeEntry(slot, [1, 2], [-1, 1])], [q.TreeEntry(slot, [1], [-2])],
                [q.TreeEntry(slot, [10 ** 6], [-1])]):
        with pytest.raises(q.StepError):
            engine.step_tree(bad)
    with pytest.raises(q.StepError):
        engine.keep({slot: []})
    with pytest.raises(q.CacheError):
        engine.step_tree([q.TreeEntry(slot, [1], [-1]), q.TreeEntry(slot, [1], [-1])])
    with pytest.raises(q.CacheFull):
        engine.step_tree([q.TreeEntry(slot, [1] * 130, [-1] * 130)])
    engine.step_tree([q.TreeEntry(other, [4], [-1]), q.TreeEntry(slot, [5, 6, 7], [-1, 0, 0])])
    for bad in ({slot: [0]}, {slot: [0], other: [], 99: []}, {slot: [0, 0], other: []}, {slot: [1], other: []}, {slot: [0, 1, 2], other: []}, {slot: [3], other: [0]}):
        with pytest.raises(q.StepError):
            engine.keep(bad)
    with pytest.raises(q.StepError):
        engine.step([q.StepEntry(slot, [1])])
    with pytest.raises(q.StepError):
        engine.step_tree([q.TreeEntry(slot, [1], [-1])])
    engine.release(other)                                                # a sequence may end meanwhile
    engine.keep({slot: [0, 2]})
    assert engine.length(slot) == 4
    engine.step([q.StepEntry(slot, [1])])
    engine.step_tree([q.TreeEntry(slot, [1] * 100, list(range(-1, 99)))])
    engine.keep({slot: []})
    assert engine.length(slot) == 5 and engine.cache.pages_held() == 1
    engine.release(slot)
    with pytest.raises(ValueError):
        engine_of(tmp_path, "B", "float32", "int4")


def test_models_that_have_no_such_cache(tmp_path):
    import qwen3_b200 as q
    from lagulorn_cases import CASES
    config = q.config_from_dict(dict(CASES["A"]))
    with pytest.raises(ValueError):
        q.Engine.from_random(config, 1, max_tokens=256, cache_dtype="float8")
    engine = q.Engine.from_random(config, 1, max_tokens=256)
    slot = engine.new_sequence()
    with pytest.raises(q.StepError):
        engine.step_tree([q.TreeEntry(slot, [1], [-1])])
