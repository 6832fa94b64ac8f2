"""Which decode mode an engine's steps run in, and what they leave to the model (CPU)."""
from types import SimpleNamespace

import pytest

from test_model_gpu import _tiny


def _engine(model, on, runner=None):
    from qwen3_engine_from_scratch_amd.engine import Engine

    # as Engine.__init__ leaves the mode
    model._invariant = on
    e = SimpleNamespace(model=model, runner=runner, batch_invariant=on,
                        _invariant_set=model._invariant_set)
    e.mode = lambda: Engine._mode(e)
    return e


def test_whose_mode_a_step_runs_in():
    model, _, _ = _tiny(layers=1, vocab=256, hidden=128, inter=128, hq=1, hkv=1)
    assert model.decode_batch_invariant is False
    eager, captured = _engine(model, False), _engine(model, False, runner=object())
    exact = _engine(model, True)
    # engines made later change nothing for those before them
    assert model.decode_batch_invariant is True
    assert (eager.mode(), captured.mode(), exact.mode()) == (False, False, True)
    # a program that sets the mode is followed by eager engines, not by captured ones
    model.decode_batch_invariant = True
    assert (eager.mode(), captured.mode(), exact.mode()) == (True, False, True)
    late = _engine(model, False)
    assert late.mode() is False and eager.mode() is True
    model.decode_batch_invariant = 0
    assert (eager.mode(), captured.mode(), exact.mode(), late.mode()) == (False, False, False, False)


def test_a_mode_ends_with_its_step():
    model, _, _ = _tiny(layers=1, vocab=256, hidden=128, inter=128, hq=1, hkv=1)
    eager = _engine(model, False)
    model.decode_batch_invariant = True
    with model.decode_mode(False):
        assert model.decode_batch_invariant is False
    assert model.decode_batch_invariant is True and eager.mode() is True
    with pytest.raises(RuntimeError, match="a step"):
        with model.decode_mode(False):
            raise RuntimeError("a step that fails")
    assert model.decode_batch_invariant is True
