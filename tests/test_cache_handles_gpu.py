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


def test_more_forks_than_one_launch_holds(gpu):
    """700 rows forked from 20, some several times, across the launches' borders."""
    from qwen3_engine_from_scratch_amd.kernels.paged_cache import fork_pages_hip
    from test_paged_cache_gpu import _bits, _pool

    announce("700 forks of 20 rows")
    g = torch.Generator().manual_seed(3)
    bs, width, n = 16, 5, 700
    k, v = _pool(gpu, 900, 1, 2, bs, 128, seed=6)
    table = torch.randint(0, 900, (n + 40, width), generator=g).to(torch.int32)
    table[:20] = torch.randperm(100, generator=g).view(20, width).to(torch.int32)  # the parents'
    seq = torch.randint(0, 60, (n + 40,), generator=g).to(torch.int32)
    src = torch.randint(0, 20, (n,), generator=g).tolist()
    dst = (20 + torch.randperm(n + 20, generator=g)[:n]).tolist()
    tokens = torch.randint(0, width * bs + 1, (n,), generator=g).tolist()
    tokens[239:242] = [17, 16, 15]  # around the first launch's end
    new = (100 + torch.randperm(800, generator=g)[:n]).tolist()
    wk, wv, wt, ws = k.clone(), v.clone(), table.clone(), seq.clone()
    for a, b, m, p in zip(src, dst, tokens, new):
        full, rest = m // bs, m % bs
        wt[b] = -1
        wt[b, :full] = table[a, :full]
        ws[b] = m
        if rest:
            wt[b, full] = p
            for x in (wk, wv):
                x[p] = 0
                x[p, :, :, :rest] = x[int(table[a, full]), :, :, :rest]
    dt, ds = table.to(gpu), seq.to(gpu)
    fork_pages_hip(k, v, dt, ds, src, dst, tokens, new)
    torch.cuda.synchronize()
    assert torch.equal(dt.cpu(), wt) and torch.equal(ds.cpu(), ws)
    assert torch.equal(_bits(k), _bits(wk)) and torch.equal(_bits(v), _bits(wv))
