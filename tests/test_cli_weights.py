"""The command line's options of weights and devices, as far as they need no GPU."""
import json

import pytest

import qwen3_b200 as q
from helpers import tiny
from qwen3_b200.cli import chat


def config_file(tmp_path, cfg):
    path = tmp_path / "config.json"
    path.write_text(json.dumps(cfg))
    return str(path)


class Made(Exception):
    pass


def made(*args, **kwargs):
    raise Made(kwargs)


@pytest.fixture(autouse=True)
def current(monkeypatch):
    """The devices that were made the current one."""
    import torch
    seen = []
    monkeypatch.setattr(torch.cuda, "set_device", seen.append)
    return seen


def test_a_model_that_takes_no_8_bit_weights_is_a_usage_error(tmp_path, monkeypatch, capsys):
    from dozazen_cases import case
    monkeypatch.setattr(q.Engine, "from_random", made)
    args = ["--random-weights", "1", "--tokens", "1,2", "--max-context", "64", "--config"]
    with pytest.raises(SystemExit):
        chat.main(args + [config_file(tmp_path, case("A")), "--weight-dtype", "int8"])
    assert "--weight-dtype" in capsys.readouterr().err
    with pytest.raises(Made):
        chat.main(args + [config_file(tmp_path, case("A"))])
    with pytest.raises(Made) as asked:
        chat.main(args + [config_file(tmp_path, tiny("A")), "--weight-dtype", "int8"])
    assert asked.value.args[0]["weight_dtype"] == "int8"


@pytest.mark.parametrize("gpu", [0, 1, 3])
def test_the_device_asked_for_is_the_current_one_when_the_engine_is_made(tmp_path, monkeypatch, current, gpu):
    """Kernels go to the current device's streams, wherever the tensors lie."""
    monkeypatch.setattr(q.Engine, "from_random", lambda *args, **kwargs: made(current=list(current), **kwargs))
    with pytest.raises(Made) as asked:
        chat.main(["--random-weights", "1", "--tokens", "1,2", "--max-context", "64", "--gpu", str(gpu), "--config", config_file(tmp_path, tiny("A"))])
    assert asked.value.args[0]["current"] == [gpu] and asked.value.args[0]["device"] == f"cuda:{gpu}"
