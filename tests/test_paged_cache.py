"""Page operations refuse bad plans before anything is launched; the pool's count of
holders (CPU)."""
import ctypes

import pytest
import torch

from qwen3_engine_from_scratch_amd import _lib

FAKE = 1 << 20


def _a(*v):
    return (ctypes.c_int32 * len(v))(*v)


def _copy(src=(1, 2), dst=(3, 4), tokens=None, n=2, k=FAKE, v=FAKE, be=65536, se=128, bs=16, nb=8):
    return _lib.load().qwen3_page_copy_bf16(k, v, be, se, bs, nb, src and _a(*src), dst and _a(*dst),
                                            tokens and _a(*tokens), n, None)


@pytest.mark.parametrize("code,over", [
    (-1, dict(k=None)), (-1, dict(v=None)), (-1, dict(n=-1)), (-1, dict(src=None)),
    (-1, dict(dst=None)), (-1, dict(be=0)), (-1, dict(be=65536 + 128)), (-1, dict(bs=0)),
    (-1, dict(nb=0)), (-1, dict(se=0)), (-2, dict(k=FAKE + 2)), (-2, dict(se=4, be=64)),
    (-1, dict(src=(1, 8))), (-1, dict(src=(-1, 2))), (-1, dict(dst=(3, 8))),
    (-1, dict(dst=(3, -2))), (-1, dict(dst=(3, 3))), (-1, dict(dst=(2, 4))),
    (-1, dict(src=(1, 1), dst=(1, 4))), (-1, dict(tokens=(16, 17))), (-1, dict(tokens=(-1, 3))),
    (0, dict(n=0)), (-1, dict(n=9)), (-3, dict(be=1 << 32)),
])
def test_copy_refuses(code, over):
    assert _copy(**over) == code, _lib.load().qwen3_attn_last_error()


def _fork(src=(0, 1), dst=(2, 3), tokens=(20, 32), new=(5, -1), n=2, bt=FAKE, sl=FAKE, stride=8,
          rows=4, pages=8):
    return _lib.load().qwen3_page_fork_bf16(FAKE, FAKE, 65536, 128, 16, 8, bt, stride, rows, pages,
                                            sl, src and _a(*src), dst and _a(*dst),
                                            tokens and _a(*tokens), new and _a(*new), n, None)


@pytest.mark.parametrize("over", [
    dict(bt=None), dict(sl=None), dict(src=None), dict(dst=None), dict(tokens=None),
    dict(new=None), dict(n=-1), dict(stride=7), dict(rows=0), dict(pages=0), dict(src=(0, 4)),
    dict(dst=(2, -1)), dict(dst=(2, 2)), dict(dst=(1, 3)), dict(tokens=(20, 129)),
    dict(tokens=(-1, 0)), dict(new=(8, 0)), dict(new=(-1, 0)), dict(tokens=(20, 33), new=(5, 5)),
])
def test_fork_refuses(over):
    assert _fork(**over) == -1, _lib.load().qwen3_attn_last_error()


def _move(src=(1, 2), dst=(3, 4), n=2, bt=FAKE, stride=8):
    return _lib.load().qwen3_page_move_bf16(FAKE, FAKE, 65536, 128, 16, 8, bt, stride, 4, 8,
                                            src and _a(*src), dst and _a(*dst), n, None)


@pytest.mark.parametrize("over", [
    dict(bt=None), dict(src=None), dict(n=-1), dict(stride=7), dict(src=(1, 1)), dict(dst=(3, 3)),
    dict(dst=(3, 1)), dict(src=(1, 9)),
])
def test_move_refuses(over):
    assert _move(**over) == -1, _lib.load().qwen3_attn_last_error()


def test_nothing_to_do_is_no_error():
    assert _fork(n=0) == 0 and _move(n=0) == 0


def test_wrappers_refuse():
    from qwen3_engine_from_scratch_amd.kernels.paged_cache import (copy_pages_hip, fork_pages_hip,
                                                                  move_pages_hip)

    k = torch.zeros(4, 1, 2, 16, 128, dtype=torch.bfloat16)
    t = torch.zeros(2, 3, dtype=torch.int32)
    s = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: copy_pages_hip(k, k.clone(), [0], [1]),
                 lambda: fork_pages_hip(k, k.clone(), t, s, [0], [1], [3], [2]),
                 lambda: move_pages_hip(k, k.clone(), t, [0], [1])):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    for call in (lambda: copy_pages_hip(k, k, [0], [1, 2]),
                 lambda: copy_pages_hip(k, k, [0], [1], [1, 2]),
                 lambda: copy_pages_hip(k, k, [2 ** 32], [1]),
                 lambda: fork_pages_hip(k, k, t, s, [0], [1], [3], [])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        copy_pages_hip(k, k, [0.5], [1])
    for bad in (k.float(), k[:, :, :, ::2], k[0]):
        with pytest.raises(AssertionError):
            copy_pages_hip(bad, bad, [0], [1])
    with pytest.raises(AssertionError):
        move_pages_hip(k, k, t.long(), [0], [1])
    with pytest.raises(AssertionError):
        fork_pages_hip(k, k, t, s[:1], [0], [1], [3], [2])


def test_holders_are_counted():
    from qwen3_engine_from_scratch_amd.PagedKVcache import KVCachePool

    pool = KVCachePool(6, 1, 16, 1, 128, device="cpu", dtype=torch.bfloat16, max_seq_len=64,
                       max_requests=4)
    a = pool.take_blocks(3)
    pool.share(a[:2])
    pool.share(a[:1])
    assert pool.is_shared(a[0]) and pool.is_shared(a[1]) and not pool.is_shared(a[2])
    pool.free(a)
    assert pool.free_block_ids == [0, 1, 2, a[2]]
    pool.free(a[:2])
    assert pool.free_count == 5 and pool.is_shared(a[0]) is False
    pool.free(a[:1])
    assert sorted(pool.free_block_ids) == list(range(6))


def test_freed_handles_and_mixed_pools_are_refused():
    from qwen3_engine_from_scratch_amd.PagedKVcache import KVCachePool, PagedKVCache, fork_caches

    pools = [KVCachePool(6, 1, 16, 1, 128, device="cpu", dtype=torch.bfloat16, max_seq_len=64,
                         max_requests=4) for _ in range(2)]
    a, b = (PagedKVCache(p) for p in pools)
    with pytest.raises(ValueError, match="several pools"):
        fork_caches([a, b])
    with pytest.raises(ValueError, match="another pool"):
        pools[0].compact([b])
    with pytest.raises(ValueError, match="cannot fork"):
        a.fork(1)
    a.free()
    with pytest.raises(ValueError, match="freed"):
        a.fork()
    with pytest.raises(ValueError, match="cannot keep"):
        a.truncate(0)
    assert all(p.free_count == 6 for p in pools)


def test_rows_and_requests_that_cannot_be_extended_are_refused():
    from types import SimpleNamespace

    from qwen3_engine_from_scratch_amd.PagedKVcache import KVCachePool, PagedKVCache
    from qwen3_engine_from_scratch_amd.engine import Engine, GenRequest
    from qwen3_engine_from_scratch_amd.model import Qwen3ForCausalLM

    pools = [KVCachePool(6, 1, 16, 1, 128, device="cpu", dtype=torch.bfloat16, max_seq_len=64,
                         max_requests=4) for _ in range(2)]
    a, b = (PagedKVCache(p) for p in pools)
    ids = torch.zeros(2, 3, dtype=torch.long)
    for caches in ([a, a], [a, b]):
        with pytest.raises(ValueError, match="handle of its own"):
            Qwen3ForCausalLM.extend(SimpleNamespace(), ids, caches)
    engine = SimpleNamespace(pool=pools[0], prefill_chunk=None)
    with pytest.raises(ValueError, match="token of its own"):
        Engine._prefill_pieces(engine, [GenRequest(0, [], 4, prefix=a)])
    with pytest.raises(ValueError, match="another pool"):
        Engine._prefill_pieces(engine, [GenRequest(0, [1], 4, prefix=b)])
    assert all(p.free_count == 6 for p in pools)
