"""Models that engines already run keep their weights as they are."""

from __future__ import annotations

import numpy as np
import pytest

from helpers import TINY_B, device_model, make_model_folder, random_tokens
from test_float8_engine import SHAPE, make_engine
from llm_inference_b200.engine.loading import load_model

gpu = pytest.mark.gpu


def test_a_model_that_something_runs_is_refused(tmp_path):
    class Runner:
        pass

    model = load_model(make_model_folder(tmp_path / "m", TINY_B, seed=3), "bfloat16", "cpu")
    runner = Runner()
    model.runners.add(runner)
    with pytest.raises(ValueError, match="engine"):
        model.to_float8()
    assert model.weights is None and not any(block.mixer.float8 for block in model.blocks)
    del runner  # given up without being closed
    model.to_float8()
    assert model.weights == "float8"


@gpu
def test_weights_under_an_open_engine_stay():
    """Captured steps hold the weights' addresses: laying them out anew under an engine that runs them is refused, and done once it is closed."""
    model, _, _ = device_model(SHAPE, 7, "bfloat16", 0.05)
    prompt = random_tokens(np.random.default_rng(4), 500, 20)
    with make_engine(model) as engine:
        before = engine.generate(prompt, max_new_tokens=8)
        with pytest.raises(ValueError, match="engine"):
            model.to_float8()
        assert model.weights is None and engine.generate(prompt, max_new_tokens=8) == before
    model.to_float8()
    assert model.weights == "float8"
    with make_engine(model, weights="float8") as engine:
        assert len(engine.generate(prompt, max_new_tokens=8)) == 8
