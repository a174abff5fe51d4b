"""Which layers and models take a cache in 8 bits and steps with drafted tokens: those whose rows hang on nothing but their own sequence's cached rows."""
import dataclasses

import pytest

import qwen3_b200 as q
from helpers import tiny

ROPE = q.PartSpec("rope", {"head_dim": 16, "theta": 1e4, "max_positions": 128})
NORM = q.PartSpec("rms_norm", {"size": 16, "eps": 1e-6})


def plan_with(**params):
    """A Qwen3 plan whose attention has further options."""
    plan = q.config_from_dict(tiny("A")).plan()
    layers = [dataclasses.replace(s, mixer=q.PartSpec(s.mixer.kind, dict(s.mixer.params, **params))) for s in plan.layers]
    return dataclasses.replace(plan, layers=layers)


TAKEN = [{}, {"position": None}, {"qk_norm": None}, {"head_gate": True}, {"out_bias": True}, {"norm_once": True, "qk_norm": None}]
REFUSED = [{"window": 32}, {"chunk": 32}, {"value_dim": 32}, {"bias": True}, {"softcap": 30.0}, {"sink": True}, {"learned_sink": True},
           {"value_heads": 1}, {"out_float32": True}, {"window": 32, "keep_first": 2}, {"value_mix": "first"}, {"value_mix": "blend"},
           {"conv_taps": 4}, {"conv_taps": 1}, {"window": 64, "pool": 16}, {"tied_values": True}, {"value_position": ROPE}, {"out_gate": True},
           {"norm_once": True}, {"norm_once": True, "temperature": {"coef": 0.1, "every": 8}}, {"distance_bias": 64}, {"shared_kv": True}]


@pytest.mark.parametrize("options", TAKEN)
def test_attention_that_takes_rows(options):
    assert all(b.mixer.takes_rows() for b in q.build_model(plan_with(**options)).blocks)


@pytest.mark.parametrize("options", REFUSED, ids=lambda o: "-".join(o))
def test_attention_that_does_not(options):
    """Every option that makes a row from more than its own projection, or reads the cache in another way than over all keys."""
    assert not any(b.mixer.takes_rows() for b in q.build_model(plan_with(**options)).blocks)


def shifted_plan(**params):
    """A plan of plain attention in blocks that mix every row with the one before it, and keep the last one of a sequence."""
    plan = plan_with(**params)
    block = q.PartSpec("shift_sandwich", {"norm": plan.final_norm, "hidden_size": plan.hidden_size})
    return dataclasses.replace(plan, layers=[dataclasses.replace(s, block=block) for s in plan.layers], residual_dtype="float32")


def test_a_model_of_plain_attention_takes_both():
    model = q.build_model(plan_with())
    assert model.takes_rows() and model.takes_trees()


def test_a_block_that_keeps_a_row_takes_no_drafted_tokens():
    model = q.build_model(shifted_plan())
    assert all(n.block_state for n in model.cache_needs()) and model.takes_rows() and not model.takes_trees()


def test_a_mixer_that_keeps_a_state_takes_neither():
    """Also where the mixer itself says that it takes rows."""
    model = q.build_model(plan_with())
    need = model.blocks[1].mixer.cache_need()
    model.blocks[1].mixer.cache_need = lambda: dataclasses.replace(need, state_shape=(7,))
    assert model.blocks[1].mixer.takes_rows() and not model.takes_rows() and not model.takes_trees()


def test_a_layer_on_another_layers_cache_takes_neither():
    plan = plan_with()
    last = plan.layers[1]
    shared = q.PartSpec(last.mixer.kind, dict(last.mixer.params, shared_kv=True))
    model = q.build_model(dataclasses.replace(plan, layers=[plan.layers[0], dataclasses.replace(last, mixer=shared, cache_from=0)]))
    assert not model.takes_rows() and not model.takes_trees()
