"""What the engine and the model refuse about shared prefixes and log probabilities (CPU)."""
from types import SimpleNamespace

import pytest
import torch


def _model(vocab=8):
    return SimpleNamespace(config=SimpleNamespace(max_position_embeddings=64, vocab_size=vocab),
                           lm_head=SimpleNamespace(weight=torch.zeros(1)))


@pytest.mark.parametrize("kw", [{"batch_invariant": True}, {"max_batch": 1025}])
def test_engine_options_that_exclude_each_other(kw):
    from qwen3_engine_from_scratch_amd.engine import Engine

    with pytest.raises(ValueError, match="share_prefixes"):
        Engine(_model(), SimpleNamespace(), share_prefixes=True, **kw)


def test_model_in_the_batch_invariant_mode():
    from qwen3_engine_from_scratch_amd.model import Qwen3ForCausalLM

    with pytest.raises(ValueError, match="batch-invariant"):
        Qwen3ForCausalLM.reserve_shared_workspace(SimpleNamespace(decode_batch_invariant=True), 4,
                                                  SimpleNamespace())


@pytest.mark.parametrize("vocab,n", [(1000, 65), (1000, -1), (8, 9)])
def test_more_alternatives_than_there_are(vocab, n):
    """Refused before anything runs, whichever request of the list asks."""
    from qwen3_engine_from_scratch_amd.engine import Engine, GenRequest

    engine = SimpleNamespace(model=_model(vocab))
    reqs = [GenRequest(0, [1], 2), GenRequest(1, [1], 2, logprobs=n)]
    with pytest.raises(ValueError, match="request 1: logprobs"):
        Engine.generate(engine, reqs)
    assert reqs[0].output_ids == []


@pytest.mark.parametrize("prompt", [[], [1] * 65])
def test_prompts_that_cannot_be_scored(prompt):
    from qwen3_engine_from_scratch_amd.engine import Engine

    def no_step(*args):
        raise AssertionError("a step was run")

    engine = SimpleNamespace(model=_model())
    engine.model.prefill_logits = no_step
    engine._check_positions = lambda n: Engine._check_positions(engine, n)
    with pytest.raises(ValueError):
        Engine.score(engine, [[1, 2], prompt])


def test_a_prefill_that_fails_takes_its_log_probabilities_back():
    from qwen3_engine_from_scratch_amd.engine import Engine, GenRequest

    def pieces(reqs):
        for r in reqs:
            r.cache = SimpleNamespace(free=lambda: None)
        Engine._take(reqs[0], (7, -0.5, [(7, -0.5)]))
        raise RuntimeError("OOM: a step")

    r = GenRequest(0, [1, 2, 3], 4, logprobs=1, output_ids=[5], output_logprobs=[-1.0],
                   output_top=[[(5, -1.0)]])
    engine = SimpleNamespace(prefill_chunk=2, _prefill_pieces=pieces)
    with pytest.raises(RuntimeError, match="OOM"):
        Engine._prefill(engine, [r])
    assert (r.output_ids, r.output_logprobs, r.output_top) == ([5], [-1.0], [[(5, -1.0)]])
    Engine._take(r, (6, -0.25, []))
    Engine._take(r, 9)  # (a request that does not ask)
    assert r.output_ids == [5, 6, 9] and r.output_logprobs == [-1.0, -0.25]
