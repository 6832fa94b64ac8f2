"""Engine.score refuses prompts with ids that are no tokens before a step is run (CPU)."""
from types import SimpleNamespace

import pytest


@pytest.mark.parametrize("prompt", [[-1], [3, -1, 2], [8], [1, 2, 1 << 40], [0, -100]])
def test_ids_outside_the_vocabulary(prompt):
    from qwen3_engine_from_scratch_amd.engine import Engine

    def no_step(*args):
        raise AssertionError("a step was run")

    engine = SimpleNamespace(model=SimpleNamespace(config=SimpleNamespace(vocab_size=8),
                                                   prefill_logits=no_step),
                             _check_positions=lambda n: None)
    with pytest.raises(ValueError, match="vocabulary"):
        Engine.score(engine, [[1, 2], prompt])
