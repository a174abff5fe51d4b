"""Which layers and models take weights in 8-bit integers: pre-norm blocks whose sublayers read their input through such products alone."""
import dataclasses

import pytest
import torch

import qwen3_b200 as q
from helpers import tiny
from test_takes_rows import plan_with, shifted_plan


def plan_with_ff(**params):
    plan = q.config_from_dict(tiny("A")).plan()
    layers = [dataclasses.replace(s, feed_forward=q.PartSpec(s.feed_forward.kind, dict(s.feed_forward.params, **params))) for s in plan.layers]
    return dataclasses.replace(plan, layers=layers)


@pytest.mark.parametrize("plan", [plan_with(), plan_with(window=32), plan_with(out_gate=True), plan_with(bias=True, out_bias=True), plan_with(sink=True),
                                  plan_with(conv_taps=4), plan_with_ff(activation="gelu_tanh"), plan_with_ff(activation="clamped")])
def test_models_that_take_them(plan):
    model = q.build_model(plan)
    names = model.eight_bit_names()
    specs = model.weight_specs()
    assert model.takes_eight_bit() and names <= set(specs)
    assert {n for n in specs if len(specs[n].shape) == 2 and specs[n].role == "matrix" and ".layers." in n} == names


def test_models_that_do_not():
    other = dataclasses.replace(plan_with(), layers=[dataclasses.replace(s, feed_forward=q.PartSpec(
        "dense_mlp", {"hidden_size": 64, "intermediate_size": 128})) for s in plan_with().layers])
    for plan in (plan_with(head_gate=True), shifted_plan(), other):
        model = q.build_model(plan)
        assert not model.takes_eight_bit()
        with pytest.raises(ValueError, match="8 bits"):
            model.bind({}, torch.float32, "cpu", eight_bit=True)


def test_a_weight_type_that_there_is_not():
    for make in (lambda: q.Engine.from_random(q.config_from_dict(tiny("A")), 1, weight_dtype="int4"), lambda: q.Engine.from_folder("nowhere", weight_dtype="fp8")):
        with pytest.raises(ValueError, match="weight_dtype"):
            make()


def test_rows_in_8_bits_are_refused_on_the_host():
    from qwen3_b200.csrc import ops
    with pytest.raises(ops.KernelError):
        ops.Int8Rows(torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4))
    with pytest.raises(ops.KernelError):
        ops.Int8Rows.empty(4, 64, "cpu")
