"""Cache handles at the limits of their pool, on the device: what the pages hold after a
give-back in a full pool."""
import pytest
import torch

from conftest import announce
from test_paged_cache_gpu import _all_free, _append, _cache_pool, _holds

pytestmark = pytest.mark.gpu


def test_truncate_in_a_full_pool(gpu):
    from qwen3_engine_from_scratch_amd.PagedKVcache import PagedKVCache

    announce("truncate into a shared page, no block free")
    pool = _cache_pool(gpu, blocks=5, rows=3)
    a = PagedKVCache(pool)
    a0 = _append(a, 48, 1)
    b = a.fork()
    b0 = _append(b, 30, 2)
    assert pool.free_count == 0
    b.truncate(40)
    _holds(b, [[x[:, :, :40] for x in a0]])
    _holds(a, [a0])
    for layer in range(2):  # the slots behind are zero, as a fresh page's
        for x in (pool.k_buffer, pool.v_buffer):
            assert not x[b.block_table[2], layer, :, 8:].any()
    assert pool.free_count == 1 and not b0[0].isnan().any()
    b1 = _append(b, 20, 3)
    _holds(b, [[x[:, :, :40] for x in a0], b1])
    _holds(a, [a0])
    a.free()
    b.free()
    _all_free(pool)
