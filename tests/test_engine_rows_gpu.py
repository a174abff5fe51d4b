"""Engines over a cache in 8 bits and with drafted tokens: models that do not take them, and what a step may not leave behind."""
import pytest

import qwen3_b200 as q
from helpers import tiny
from test_takes_rows import plan_with

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
