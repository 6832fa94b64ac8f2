"""An engine's steps run in their own decode mode and leave the model's as it was; an eager
engine follows a program that sets it."""
import pytest
import torch

from conftest import announce
from test_model_gpu import _pool, _tiny

pytestmark = pytest.mark.gpu


def test_the_models_mode_after_a_step(gpu):
    from qwen3_engine_from_scratch_amd.engine import Engine, GenRequest

    model, _, cfg = _tiny(seed=21)
    model = model.to(gpu)
    g = torch.Generator().manual_seed(3)
    asks = [torch.randint(0, cfg.vocab_size, (20 + i,), generator=g).tolist() for i in range(3)]
    pool = _pool(cfg, gpu, blocks=90, max_requests=48)

    def run(engine, told):
        engine.generate([GenRequest(i, a, 4, logprobs=1 if told else None) for i, a in enumerate(asks)])
        return model._ws_mode

    announce("an eager and a captured engine, the model's mode set between their steps")
    eager = Engine(model, pool, max_batch=4, use_graph=False)
    captured = Engine(model, pool, max_batch=4)
    for on in (True, False, True):
        model.decode_batch_invariant = on  # after the engines were made
        for told in (True, False):
            assert run(eager, told) is on
            assert model.decode_batch_invariant is on
        assert run(captured, True) is False  # as it was captured
        assert model.decode_batch_invariant is on
    announce("an engine of the other mode made later")
    exact = Engine(model, pool, max_batch=4, use_graph=False, batch_invariant=True)
    model.decode_batch_invariant = False
    kept = Engine(model, pool, max_batch=4, use_graph=False, batch_invariant=True)
    assert run(exact, False) is False and run(kept, False) is True and run(kept, True) is True
    late = Engine(model, pool, max_batch=4, use_graph=False)
    assert run(kept, False) is True and run(late, True) is False
    assert model.decode_batch_invariant is False
    for e in (eager, captured, exact, kept, late):
        e.close()
    assert pool.free_count == pool.total_blocks


def test_sharing_follows_no_program_into_the_batch_invariant_mode(gpu):
    """Refused, not run in another mode than the program asked for; the engine goes on when
    the mode is taken back."""
    from qwen3_engine_from_scratch_amd.engine import Engine, GenRequest

    model, _, cfg = _tiny(seed=22)
    model = model.to(gpu)
    pool = _pool(cfg, gpu, blocks=90, max_requests=48)
    engine = Engine(model, pool, max_batch=4, use_graph=False, share_prefixes=True)
    prefix = engine.cache_prefix(list(range(40)))

    def reqs():
        return [GenRequest(i, [7, 8, i], 3, prefix=prefix) for i in range(3)]

    announce("sharing while the model is set batch-invariant")
    engine.generate(reqs())
    model.decode_batch_invariant = True
    with pytest.raises(ValueError, match="batch-invariant"):
        engine.generate(reqs())
    assert model.decode_batch_invariant is True
    model.decode_batch_invariant = False
    again = reqs()
    engine.generate(again)
    assert all(len(r.output_ids) == 3 for r in again)
    prefix.free()
