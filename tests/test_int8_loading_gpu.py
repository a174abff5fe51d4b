"""What loading a model with 8-bit weights takes from the device, and what it keeps."""
import gc

import pytest
import torch

import qwen3_b200 as q
from helpers import tiny

pytestmark = pytest.mark.gpu
WIDE = dict(num_hidden_layers=6, hidden_size=1024, intermediate_size=4096, torch_dtype="bfloat16")


def settle():
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def matrices(model):
    return [w for b in model.blocks for w in (b.mixer.w_qkv, b.mixer.w_o, b.feed_forward.w_gate_up, b.feed_forward.w_down)]


def test_nothing_but_the_codes_is_kept_of_a_checkpoint(tmp_path):
    """The device gives the arena, one layer as it is stored and the staging buffers, and of these the arena alone is kept: codes and scales lie in it.  (64 MB:
    staging, the step's buffers and the allocator's pieces.)"""
    config = q.config_from_dict(tiny("B", **WIDE))
    folder = str(tmp_path / "model")
    q.write_random_model(folder, config, 2)
    q.Engine.from_folder(folder, dtype="bfloat16", max_tokens=64, max_seq_len=64, weight_dtype="int8")     # (status words, kernels' memory)
    settle()
    before, held = torch.cuda.memory_reserved(), torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    engine = q.Engine.from_folder(folder, dtype="bfloat16", max_tokens=64, max_seq_len=64, weight_dtype="int8")
    arena, layer = engine.weights_arena, 2 * sum(w.rows * w.width for w in matrices(engine.model)[:4])
    assert torch.cuda.max_memory_reserved() - before <= arena.numel() + layer + (128 << 20)
    settle()
    unused = (torch.cuda.memory_reserved() - torch.cuda.memory_allocated()) - (before - held)
    assert unused <= 64 << 20, unused
    lo, hi = arena.data_ptr(), arena.data_ptr() + arena.numel()
    for w in matrices(engine.model):
        for t in (w.codes, w.scales):
            assert lo <= t.data_ptr() and t.data_ptr() + t.numel() * t.element_size() <= hi
    codes = sum(w.rows * (w.stride + 4) for w in matrices(engine.model))
    embeddings = 2 * 2 * config.vocab_size * config.hidden_size
    assert arena.numel() <= codes + embeddings + (1 << 20)


@pytest.mark.parametrize("name", ["A", "C", "D"])
@pytest.mark.parametrize("storage", ["bfloat16", "float32"])
def test_codes_in_the_arena_are_those_of_the_stored_matrices(tmp_path, name, storage):
    """Widths that leave room behind every row, and matrices that are made of several."""
    from helpers import make_folder
    from qwen3_b200.csrc import ops
    folder, _ = make_folder(tmp_path, tiny(name), seed=4, storage=storage)
    got = q.Engine.from_folder(folder, dtype="float32", max_tokens=64, weight_dtype="int8").model
    plain = q.Engine.from_folder(folder, dtype="float32", max_tokens=64).model
    for a, b in zip(matrices(got), matrices(plain)):
        want = ops.quantize_rows(b, ops.Int8Rows.empty(*b.shape, "cuda"))
        assert torch.equal(a.codes, want.codes) and torch.equal(a.scales, want.scales)


def test_drawn_weights_are_given_back_while_they_are_quantised(monkeypatch):
    """When the engine's own memory is taken, the device holds the codes and the embeddings; at no time much more than all matrices as drawn."""
    config = q.config_from_dict(tiny("B", **WIDE))
    held = []
    built = q.Engine.__init__

    def init(self, model, *args, **kwargs):
        held.append((torch.cuda.memory_allocated(), torch.cuda.max_memory_allocated()))
        built(self, model, *args, **kwargs)
    monkeypatch.setattr(q.Engine, "__init__", init)
    q.Engine.from_random(config, 3, dtype="bfloat16", max_tokens=64, max_seq_len=64, weight_dtype="int8")
    settle()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    engine = q.Engine.from_random(config, 3, dtype="bfloat16", max_tokens=64, max_seq_len=64, weight_dtype="int8")
    codes = sum(w.rows * (w.stride + 4) for w in matrices(engine.model))
    drawn = 2 * sum(w.rows * w.width for w in matrices(engine.model))
    embeddings = 2 * 2 * config.vocab_size * config.hidden_size
    now, peak = held[-1]
    assert now - before <= codes + embeddings + (8 << 20)
    assert peak - before <= drawn + embeddings + drawn // 4 + (32 << 20)


@pytest.mark.parametrize("weight_dtype", [None, "int8"])
def test_memory_that_is_still_being_written_when_the_arena_gets_it(tmp_path, weight_dtype):
    """A kernel that is queued before the load writes a tensor of the arena's size, which the program has given up: the arena is likely to be its memory."""
    from helpers import make_folder
    folder, _ = make_folder(tmp_path, tiny("B", num_hidden_layers=4, hidden_size=256, intermediate_size=1024), seed=5)
    load = lambda: q.Engine.from_folder(folder, dtype="bfloat16", max_tokens=64, max_seq_len=64, weight_dtype=weight_dtype)  # noqa: E731
    first = load()
    torch.cuda.synchronize()
    size = first.weights_arena.numel()
    for _ in range(3):
        memory = torch.empty(size, dtype=torch.uint8, device="cuda")
        torch.cuda._sleep(200_000_000)                     # 0.1 s
        memory.fill_(255)
        del memory
        engine = load()
        torch.cuda.synchronize()
        for (name, a), (_, b) in zip(parameters(first.model), parameters(engine.model)):
            assert torch.equal(a, b), name
        del engine


def parameters(model):
    out = [("embedding", model.embedding.table), ("head", model.head.weight), ("norm", model.final_norm.weight)]
    for i, w in enumerate(matrices(model)):
        out += [(f"{i} codes", w.codes), (f"{i} scales", w.scales)] if hasattr(w, "codes") else [(str(i), w)]
    return out
