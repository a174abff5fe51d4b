"""Models whose projections are not to be had in 8 bits are refused before anything is read, drawn or allocated for them."""
import pytest

import qwen3_b200 as q
from helpers import tiny


def not_reached(*args, **kwargs):
    raise AssertionError("weights were asked for")


def test_refused_before_weights_are_asked_for(tmp_path, monkeypatch):
    from dozazen_cases import case
    from qwen3_b200.engine import engine as engine_module
    config = q.config_from_dict(case("A"))
    folder = str(tmp_path / "model")
    q.write_random_model(folder, config, 1)
    for name in ("open_upload", "random_weights"):
        monkeypatch.setattr(engine_module, name, not_reached)
    with pytest.raises(ValueError, match="8 bits"):
        q.Engine.from_folder(folder, max_tokens=64, weight_dtype="int8")
    with pytest.raises(ValueError, match="8 bits"):
        q.Engine.from_random(config, 1, max_tokens=64, weight_dtype="int8")
    for taken, weight_dtype in ((q.config_from_dict(tiny("A")), "int8"), (config, None)):
        with pytest.raises(AssertionError, match="asked for"):           # (others go on to their weights)
            q.Engine.from_random(taken, 1, max_tokens=64, weight_dtype=weight_dtype)


def test_drawn_weights_are_held_by_the_model_alone(monkeypatch):
    """When the engine's own memory is taken, a matrix that was made into another one is gone."""
    import weakref
    from qwen3_b200.engine import engine as engine_module
    drawn, alive = {}, []
    plain = engine_module.random_weights

    def draw(*args, **kwargs):
        tensors = plain(*args, **kwargs)
        drawn.update({name: weakref.ref(t) for name, t in tensors.items()})
        return tensors
    monkeypatch.setattr(engine_module, "random_weights", draw)
    monkeypatch.setattr(q.Engine, "__init__", lambda self, *args: alive.extend(n for n, t in drawn.items() if t() is not None))
    q.Engine.from_random(q.config_from_dict(tiny("A")), 1, dtype="bfloat16", max_tokens=64, device="cpu")
    assert len(drawn) > 10 and not [n for n in alive if any(part in n for part in ("q_proj", "k_proj", "v_proj", "gate_proj", "up_proj"))]


def test_parts_that_do_something_else_are_not_taken_for_those_they_are_built_on():
    """A norm or a block of another formula would otherwise run with the formula of its base, without an error."""
    from qwen3_b200.parts.block import PreNormBlock
    from qwen3_b200.parts.norm import RMSNorm

    class HalvedNorm(RMSNorm):
        def __call__(self, x, out, delta=None):
            return super().__call__(x, out, delta).mul_(0.5)

    class Renamed(RMSNorm):
        pass

    class OtherBlock(PreNormBlock):
        def forward(self, residual, delta, ctx, cache):
            return super().forward(residual, delta, ctx, cache)
    model = q.build_model(q.config_from_dict(tiny("A")).plan())
    assert model.takes_eight_bit() and Renamed(64, 1e-6).takes_eight_bit()
    assert not HalvedNorm(64, 1e-6).takes_eight_bit()
    block = model.blocks[0]
    kept = block.mixer_norm
    block.mixer_norm = HalvedNorm(64, 1e-6)
    assert not model.takes_eight_bit()
    block.mixer_norm, block.__class__ = kept, OtherBlock
    assert not model.takes_eight_bit()


def test_widths_whose_sums_do_not_fit_32_bits():
    """Refused with the model, not by its first step."""
    from qwen3_b200.csrc import ops
    from qwen3_b200.parts.attention import GQAAttention
    from qwen3_b200.parts.mlp import SwiGLU
    most = ops.INT8_MAX_WIDTH
    assert SwiGLU(64, most).takes_eight_bit() and not SwiGLU(64, most + 1).takes_eight_bit() and not SwiGLU(most + 1, 64).takes_eight_bit()
    assert GQAAttention(most, 4, 2, 16, 1.0).takes_eight_bit() and not GQAAttention(most + 1, 4, 2, 16, 1.0).takes_eight_bit()
    assert not GQAAttention(64, 1024, 2, 128, 1.0).takes_eight_bit()


def test_sources_that_round_before_they_are_quantised():
    """A source of tensors that was not told of the 8 bits hands out 32-bit matrices rounded to bfloat16."""
    import types
    import torch
    model = q.build_model(q.config_from_dict(tiny("A")).plan())
    tensors = q.random_weights(model.weight_specs(), 1, dtype=torch.float32)
    for source in (types.SimpleNamespace(), types.SimpleNamespace(apart=set()), types.SimpleNamespace(apart=set(list(model.eight_bit_names())[1:])),
                   model.source_of(tensors, torch.bfloat16, "cpu")):
        with pytest.raises(ValueError, match="rounded"):
            model.bind(source, torch.bfloat16, "cpu", eight_bit=True)
    kept = model.source_of(tensors, torch.bfloat16, "cpu", eight_bit=True)
    assert {n for n, t in kept.items() if t.dtype == torch.float32} >= model.eight_bit_names()
