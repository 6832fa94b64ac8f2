"""Pages copied, forked and moved: the kernels against plain indexing (copies are bits:
equal or wrong), and fork / truncate / compact of the cache handles."""
import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu


def _pool(dev, blocks, layers, heads, bs, d, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    # any bits: NaN and infinities are copied like numbers
    return [torch.randint(-2 ** 15, 2 ** 15, (blocks, layers, heads, bs, d), generator=g,
                          device=dev, dtype=torch.int16).view(torch.bfloat16) for _ in range(2)]


def _bits(t):
    return t.view(torch.int16)


@pytest.mark.parametrize("layers,heads,bs,d", [(1, 1, 16, 128), (28, 8, 16, 128), (3, 2, 48, 64),
                                               (2, 5, 1, 8), (1, 3, 7, 24)])
def test_copy(gpu, layers, heads, bs, d):
    from qwen3_engine_from_scratch_amd.kernels.paged_cache import copy_pages_hip

    announce(f"page copies {layers} x {heads} x {bs} x {d}")
    k, v = _pool(gpu, 20, layers, heads, bs, d)
    src, dst = [3, 3, 19, 0], [7, 1, 2, 18]  # a source may serve several
    tokens = [bs, 0, bs // 2, bs - 1]
    want = [x.clone() for x in (k, v)]
    for x in want:
        for a, b, n in zip(src, dst, tokens):
            x[b] = 0
            x[b, :, :, :n] = x[a, :, :, :n]
    copy_pages_hip(k, v, src, dst, tokens)
    torch.cuda.synchronize()
    for x, w in zip((k, v), want):
        assert torch.equal(_bits(x), _bits(w))
    for x in want:
        x[5] = x[7]
    copy_pages_hip(k, v, [7], [5])
    copy_pages_hip(k, v, [], [])
    torch.cuda.synchronize()
    for x, w in zip((k, v), want):
        assert torch.equal(_bits(x), _bits(w))


def test_more_copies_than_one_launch_holds(gpu):
    from qwen3_engine_from_scratch_amd.kernels.paged_cache import copy_pages_hip, move_pages_hip

    announce("700 page copies, 700 page moves")
    k, v = _pool(gpu, 1500, 1, 2, 16, 128, seed=1)
    g = torch.Generator().manual_seed(2)
    ids = torch.randperm(1500, generator=g).tolist()
    src, dst = ids[:700], ids[700:1400]
    want = [x.clone() for x in (k, v)]
    for x in want:
        x[dst] = x[src]
    copy_pages_hip(k, v, src, dst)
    torch.cuda.synchronize()
    for x, w in zip((k, v), want):
        assert torch.equal(_bits(x), _bits(w))
    k, v = _pool(gpu, 1500, 1, 2, 16, 128, seed=3)
    want = [x.clone() for x in (k, v)]
    for x in want:
        x[dst] = x[src]
    table = torch.randint(-1, 1500, (37, 91), generator=g).to(torch.int32)
    to = torch.arange(1500, dtype=torch.int32)
    to[src] = torch.tensor(dst, dtype=torch.int32)
    expect = torch.where(table >= 0, to[table.clamp(min=0).long()], table)
    hold = torch.full((37, 100), 5, dtype=torch.int32, device=gpu)  # rows with a stride
    hold[:, :91] = table.to(gpu)
    move_pages_hip(k, v, hold[:, :91], src, dst)
    torch.cuda.synchronize()
    assert torch.equal(hold[:, :91].cpu(), expect) and (hold[:, 91:] == 5).all()
    for x, w in zip((k, v), want):
        assert torch.equal(_bits(x), _bits(w))


def test_move_leaves_foreign_entries(gpu):
    from qwen3_engine_from_scratch_amd.kernels.paged_cache import move_pages_hip

    announce("moves: entries that are no block, one move, repeated entries")
    k, v = _pool(gpu, 8, 2, 2, 16, 128)
    wk = k.clone()
    wk[0] = wk[7]
    table = torch.tensor([[7, -1, 7, 2 ** 31 - 1], [-(2 ** 31), 6, 0, 8]], dtype=torch.int32,
                         device=gpu)
    move_pages_hip(k, v, table, [7], [0])
    torch.cuda.synchronize()
    assert table.tolist() == [[0, -1, 0, 2 ** 31 - 1], [-(2 ** 31), 6, 0, 8]]
    assert torch.equal(_bits(k), _bits(wk))


@pytest.mark.parametrize("bs", [16, 48])
def test_fork(gpu, bs):
    from qwen3_engine_from_scratch_amd.kernels.paged_cache import fork_pages_hip

    announce(f"forks, blocks of {bs}")
    k, v = _pool(gpu, 40, 2, 3, bs, 128, seed=4)
    table = torch.full((300, 9), 33, dtype=torch.int32)
    table[0, :5] = torch.tensor([4, 9, 2, 30, 8])
    table[1, :2] = torch.tensor([11, -1])
    table[2, :1] = 39
    seq = torch.arange(300, dtype=torch.int32)
    src, dst = [0, 0, 0, 1, 2, 0], [5, 7, 3, 6, 4, 299]
    tokens = [4 * bs + 3, 3 * bs, 0, bs + 1, bs - 1, 9 * bs]
    new = [20, -1, -5, 21, 22, 10 ** 6]
    wk, wv, wt, ws = k.clone(), v.clone(), table.clone(), seq.clone()
    for a, b, n, m in zip(src, dst, tokens, new):
        full, rest = n // bs, n % bs
        wt[b] = -1
        wt[b, :full] = table[a, :full]
        ws[b] = n
        if rest:
            wt[b, full] = m
            old = int(table[a, full])
            if old >= 0:  # the entry -1 of row 1 names no page
                for x in (wk, wv):
                    x[m] = 0
                    x[m, :, :, :rest] = x[old, :, :, :rest]
    dt, ds = table.to(gpu), seq.to(gpu)
    fork_pages_hip(k, v, dt, ds, src, dst, tokens, new)
    torch.cuda.synchronize()
    assert torch.equal(dt.cpu(), wt) and torch.equal(ds.cpu(), ws)
    assert torch.equal(_bits(k), _bits(wk)) and torch.equal(_bits(v), _bits(wv))


def test_capture(gpu):
    from qwen3_engine_from_scratch_amd.kernels.paged_cache import copy_pages_hip, fork_pages_hip

    announce("fork and copy captured and replayed")
    k, v = _pool(gpu, 12, 2, 2, 16, 128, seed=5)
    table = torch.full((4, 4), -1, dtype=torch.int32, device=gpu)
    table[0, :2] = torch.tensor([3, 5], dtype=torch.int32)
    seq = torch.zeros(4, dtype=torch.int32, device=gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fork_pages_hip(k, v, table, seq, [0], [2], [20], [9])
        copy_pages_hip(k, v, [9], [10], [2])
    for i in range(3):
        k.view(torch.int16).add_(i + 1)
        table[0, 1] = 5 - i
        seq.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert table[2].tolist() == [3, 9, -1, -1] and seq.tolist() == [0, 0, 20, 0]
        assert torch.equal(_bits(k[9, :, :, :4]), _bits(k[5 - i, :, :, :4])) and not k[9, :, :, 4:].any()
        assert torch.equal(_bits(k[10, :, :, :2]), _bits(k[5 - i, :, :, :2])) and not k[10, :, :, 2:].any()


# ---- the handles -----------------------------------------------------------------

def _cache_pool(gpu, blocks=24, rows=12, bs=16):
    from qwen3_engine_from_scratch_amd.PagedKVcache import KVCachePool

    return KVCachePool(blocks, 2, bs, 2, 128, device=gpu, dtype=torch.bfloat16, max_seq_len=8 * bs,
                       max_requests=rows)


def _append(cache, n, seed):
    """n tokens more, all layers; returns their K as written."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pool = cache._pool
    ks = []
    for layer in range(2):
        k = torch.randn(1, 2, n, 128, generator=g, device="cuda").to(torch.bfloat16)
        cache.update(layer, k, -k)
        ks.append(k)
    cache.advance_seq_len(n)
    return ks


def _holds(cache, parts, n=None):
    """The cache's K and V of both layers are `parts` in a row, up to n tokens."""
    want_len = sum(p[0].shape[2] for p in parts) if n is None else n
    assert cache.seq_len == want_len
    assert int(cache._pool.seq_lens[cache.row_id]) == want_len
    assert cache._pool.block_table_2d[cache.row_id, :cache.num_pages].tolist() == cache.block_table
    for layer in range(2):
        want = torch.cat([p[layer] for p in parts], 2)[:, :, :want_len]
        k, v = cache.get_kv(layer)
        if want_len == 0:
            assert k is None
        else:
            assert torch.equal(k, want) and torch.equal(v, -want)


def _all_free(pool):
    assert sorted(pool.free_block_ids) == list(range(pool.total_blocks))
    assert not pool._extra_holders and len(pool._free_rows) == pool.max_requests


def test_forked_requests_go_their_own_ways(gpu):
    from qwen3_engine_from_scratch_amd.PagedKVcache import PagedKVCache, fork_caches

    announce("fork, append on both sides, fork the fork, free in any order")
    pool = _cache_pool(gpu)
    a = PagedKVCache(pool)
    a0 = _append(a, 37, 1)
    b, c, d, e = fork_caches([a, a, a, a], [37, 32, 5, 0])
    assert pool.free_count == 24 - 3 - 2  # two copies of partly filled pages, nothing else
    a1, b1 = _append(a, 6, 2), _append(b, 30, 3)
    c1, d1, e1 = _append(c, 3, 4), _append(d, 20, 5), _append(e, 2, 6)
    for cache, parts in ((a, [a0, a1]), (b, [a0, b1]), (e, [e1])):
        _holds(cache, parts)
    _holds(c, [[x[:, :, :32] for x in a0], c1])
    _holds(d, [[x[:, :, :5] for x in a0], d1])
    f = b.fork()
    f1 = _append(f, 1, 7)
    _holds(f, [a0, b1, f1])
    a.free()
    _holds(b, [a0, b1])
    b.free()
    _holds(f, [a0, b1, f1])
    _holds(c, [[x[:, :, :32] for x in a0], c1])
    for x in (e, f, c, d):
        x.free()
    _all_free(pool)


def test_truncate(gpu):
    from qwen3_engine_from_scratch_amd.PagedKVcache import PagedKVCache

    announce("truncate: own pages, shared pages, borders, nothing left")
    pool = _cache_pool(gpu)
    a = PagedKVCache(pool)
    a0 = _append(a, 60, 1)
    b = a.fork()
    b.truncate(20)          # inside a page that a holds too: a copy takes its place
    assert not pool.is_shared(b.block_table[1]) and b.block_table[1] != a.block_table[1]
    b1 = _append(b, 4, 2)
    _holds(b, [[x[:, :, :20] for x in a0], b1])
    _holds(a, [a0])
    a.truncate(32)          # a page's border: nothing copied
    _holds(a, [a0], 32)
    a1 = _append(a, 17, 3)
    _holds(a, [[x[:, :, :32] for x in a0], a1])
    a.truncate(49)          # nothing
    a.truncate(0)
    _holds(a, [a0], 0)
    _holds(b, [[x[:, :, :20] for x in a0], b1])
    with pytest.raises(ValueError):
        a.truncate(1)
    with pytest.raises(ValueError):
        b.truncate(-1)
    a.free()
    b.free()
    _all_free(pool)


def test_compact(gpu):
    from qwen3_engine_from_scratch_amd.PagedKVcache import PagedKVCache

    announce("compact: shared pages, a page of nobody's, then more tokens")
    pool = _cache_pool(gpu)
    own = pool.alloc(1)[0]  # as a captured graph's dummy page
    hs, parts = [], []
    for i in range(5):
        h = PagedKVCache(pool)
        hs.append(h)
        parts.append([_append(h, 20 + 9 * i, i)])
    f = hs[4].fork(40)
    parts_f = [[x[:, :, :40] for x in parts[4][0]]]
    hs[0].free()
    hs[2].free()
    live = [hs[1], hs[3], hs[4], f]
    used = pool.total_blocks - pool.free_count
    kept = pool.k_buffer[own].clone()
    # f's handle is not given: what it shares with hs[4] must stay
    shared = [b for b in hs[4].block_table if pool.is_shared(b)]
    pool.compact(live[:3])
    assert all(b in f.block_table for b in shared)
    moved = pool.compact(live)
    assert moved > 0 and pool.compact(live) == 0
    blocks = sorted({b for h in live for b in h.block_table})
    assert max(b for b in blocks) < used and own not in blocks
    assert torch.equal(pool.k_buffer[own], kept)
    assert sorted(pool.free_block_ids + blocks + [own]) == list(range(pool.total_blocks))
    for h, p in zip((hs[1], hs[3], hs[4]), (parts[1], parts[3], parts[4])):
        p.append(_append(h, 11, 50 + h.row_id))
        _holds(h, p)
    parts_f.append(_append(f, 9, 9))
    _holds(f, parts_f)
    for h in live:
        h.free()
    pool.free([own])
    _all_free(pool)


def test_a_pool_that_is_too_small_changes_nothing(gpu):
    from qwen3_engine_from_scratch_amd.PagedKVcache import PagedKVCache, fork_caches

    announce("fork without blocks or rows")
    pool = _cache_pool(gpu, blocks=4, rows=3)
    a = PagedKVCache(pool)
    _append(a, 60, 1)
    free, rows = list(pool.free_block_ids), list(pool._free_rows)
    with pytest.raises(RuntimeError, match="OOM"):
        a.fork()
    with pytest.raises(RuntimeError, match="OOM"):
        fork_caches([a, a, a], [0, 0, 0])
    with pytest.raises(ValueError):
        a.fork(61)
    assert pool.free_block_ids == free and pool._free_rows == rows and not pool._extra_holders
    b, c = fork_caches([a, a], [48, 0])
    assert b.block_table == a.block_table[:3]
    b.free()
    c.free()
    a.free()
    _all_free(pool)
