"""Rotary positions refuse what would lose a gradient (CPU)."""
import pytest
import torch

from qwen3_engine_from_scratch_amd.kernels.rotary import (make_rotary, rotary_embedding_decode_hip,
                                                          rotary_embedding_hip,
                                                          rotary_embedding_prefill_hip)


def _case(grad):
    t = [torch.zeros(3, h, 128, dtype=torch.bfloat16) for h in (4, 2, 2)]
    t["qkv".index(grad)].requires_grad_()
    kb = torch.zeros(2, 1, 2, 16, 128, dtype=torch.bfloat16)
    return make_rotary(128), t, torch.arange(3), kb


@pytest.mark.parametrize("grad", ["q", "k", "v"])
def test_forms_that_write_the_pool_refuse_a_gradient(grad):
    from qwen3_engine_from_scratch_amd.PagedKVcache import KVCachePool

    rot, (q, k, v), pos, kb = _case(grad)
    pool = KVCachePool(2, 1, 16, 2, 128, device="cpu", dtype=torch.bfloat16, max_seq_len=32,
                       max_requests=3)
    calls = (lambda: rotary_embedding_prefill_hip(q, k, v, pos, rot, pos, kb, kb, 0),
             lambda: rotary_embedding_decode_hip(q, k, v, rot, pool, 0))
    for call in calls:
        with pytest.raises(RuntimeError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


@pytest.mark.parametrize("grad", ["q", "k"])
def test_given_outputs_refuse_a_gradient(grad):
    rot, (q, k, _), pos, _ = _case(grad)
    for outs in (dict(q_out=torch.zeros_like(q)), dict(k_out=torch.zeros_like(k))):
        with pytest.raises(RuntimeError, match="gradient"):
            rotary_embedding_hip(q, k, pos, rot, **outs)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
            rotary_embedding_hip(q, k, pos, rot, **outs)
