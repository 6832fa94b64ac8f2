"""Handles of the paged cache that may not be used any more, and pools that run out: what is
refused, and that nothing of another request's changes (CPU; the few device writes of the
host bookkeeping run on CPU tensors)."""
from types import SimpleNamespace

import pytest
import torch

from qwen3_engine_from_scratch_amd import PagedKVcache as pc
from qwen3_engine_from_scratch_amd.PagedKVcache import KVCachePool, PagedKVCache


def _pool(blocks=6, rows=4):
    return KVCachePool(blocks, 1, 16, 1, 128, device="cpu", dtype=torch.bfloat16, max_seq_len=96,
                       max_requests=rows)


def _state(pool):
    return (list(pool.free_block_ids), list(pool._free_rows), dict(pool._extra_holders),
            pool.block_table_2d.tolist(), pool.seq_lens.tolist())


def _freed_and_its_heir():
    """A freed handle, and the request that has its row now."""
    pool = _pool()
    a = PagedKVCache(pool)
    a.reserve_slots(20)
    a.advance_seq_len(20)
    a.free()
    b = PagedKVCache(pool)
    assert b.row_id == a.row_id
    b.reserve_slots(16)
    b.advance_seq_len(5)
    return pool, a, b


def test_extend_refuses_a_freed_handle():
    from qwen3_engine_from_scratch_amd.model import Qwen3ForCausalLM

    pool, a, b = _freed_and_its_heir()
    c = PagedKVCache(pool)
    before = _state(pool)
    ids = torch.zeros(2, 3, dtype=torch.long)
    for caches in ([c, a], [a, c]):
        for lens in (None, [1, 0], [0, 0]):
            with pytest.raises(ValueError, match="freed"):
                Qwen3ForCausalLM.extend(SimpleNamespace(), ids, caches, lens)
    assert _state(pool) == before and b.block_table == [int(pool.block_table_2d[b.row_id, 0])]


@pytest.mark.parametrize("use", [
    lambda c: c.reserve_slots(3), lambda c: c.reserve_next(), lambda c: c.advance_seq_len(3),
    lambda c: c._allocate_block(),
    lambda c: c.update(0, torch.zeros(1, 1, 3, 128), torch.zeros(1, 1, 3, 128)),
    lambda c: pc.reserve_pages_bulk([c], [3]), lambda c: pc.set_seq_lens_bulk([c]),
    lambda c: pc.prefill_slot_mapping([c], 3, "cpu"),
    lambda c: pc.PageIn.reserve(SimpleNamespace(pool=c._pool, cap=8), [c], [3]),
])
def test_a_freed_handle_writes_into_no_row(use):
    pool, a, b = _freed_and_its_heir()
    before = _state(pool)
    with pytest.raises(ValueError, match="freed"):
        use(a)
    assert _state(pool) == before and a.block_table == [] and a.seq_len == 0


def test_a_second_free_gives_nothing_back_twice():
    pool = _pool()
    a, b = PagedKVCache(pool), PagedKVCache(pool)
    a.reserve_slots(20)
    b.reserve_slots(5)
    a.free()
    before = _state(pool)
    a.free()
    assert _state(pool) == before
    c, d = PagedKVCache(pool), PagedKVCache(pool)
    assert len({b.row_id, c.row_id, d.row_id}) == 3
    a.free()  # its row is c's or d's by now
    assert len(pool._free_rows) == 1


def _model(positions):
    return SimpleNamespace(config=SimpleNamespace(max_position_embeddings=positions, vocab_size=8),
                           lm_head=SimpleNamespace(weight=torch.zeros(1)))


def test_extend_refuses_positions_behind_the_tables():
    """The step that rotates knows no angle there: it would leave q and the slot unwritten."""
    from qwen3_engine_from_scratch_amd.model import Qwen3ForCausalLM

    pool = _pool()
    a, b = PagedKVCache(pool), PagedKVCache(pool)
    a.reserve_slots(38)
    a.advance_seq_len(38)
    before = _state(pool)
    ids = torch.zeros(2, 3, dtype=torch.long)
    for caches, lens in (([a, b], None), ([a, b], [3, 0]), ([b, a], [1, 3])):
        with pytest.raises(ValueError, match="positions"):
            Qwen3ForCausalLM.extend(_model(40), ids, caches, lens)
    assert _state(pool) == before
    out = Qwen3ForCausalLM.extend(_model(40), ids, [a, b], [0, 0])  # nothing to place
    assert out.shape == (2, 3, 8) and not out.any()


def test_the_engine_refuses_prompts_behind_the_tables():
    from qwen3_engine_from_scratch_amd.engine import Engine, GenRequest

    pool = _pool()
    prefix = PagedKVCache(pool)
    prefix.reserve_slots(30)
    prefix.advance_seq_len(30)
    before = _state(pool)

    def no_step(*args):
        raise AssertionError("a step was run")

    engine = SimpleNamespace(pool=pool, prefill_chunk=8, model=_model(40), _run_chunk=no_step,
                             _check_positions=lambda n: Engine._check_positions(engine, n))
    for reqs in ([GenRequest(0, [1] * 5, 4, prefix=prefix), GenRequest(1, [1] * 11, 4, prefix=prefix)],
                 [GenRequest(0, [1] * 41, 4)]):
        with pytest.raises(ValueError, match="positions"):
            Engine._prefill_pieces(engine, reqs)
    with pytest.raises(ValueError, match="positions"):
        Engine.cache_prefix(engine, [1] * 41)
    assert _state(pool) == before


def _engine(pool, fail_at):
    """An engine whose chunk step number `fail_at` finds no memory."""
    from qwen3_engine_from_scratch_amd.engine import Engine

    steps = []

    def step(caches, tokens, want_logits):
        steps.append(1)
        for c, t in zip(caches, tokens):
            c.reserve_slots(len(t))
            c.seq_len += len(t)
        if len(steps) == fail_at:
            raise RuntimeError("OOM: a step")
        return [7] * len(caches)

    return SimpleNamespace(pool=pool, prefill_chunk=8, model=_model(96), _run_chunk=step,
                           _take=Engine._take, _check_positions=lambda n: None)


@pytest.mark.parametrize("fail_at", [1, 3])
def test_a_prefix_that_fails_gives_its_row_and_pages_back(fail_at):
    from qwen3_engine_from_scratch_amd.engine import Engine

    pool = _pool()
    free, rows = sorted(pool.free_block_ids), sorted(pool._free_rows)
    with pytest.raises(RuntimeError, match="a step"):
        Engine.cache_prefix(_engine(pool, fail_at), [1] * 30)
    assert sorted(pool.free_block_ids) == free and sorted(pool._free_rows) == rows
    c = Engine.cache_prefix(_engine(pool, 9), [1] * 30)
    assert c.seq_len == 30 and not c.freed


@pytest.mark.parametrize("fail_at", [1, 2, 3])
def test_a_prefill_that_fails_leaves_nothing_behind(fail_at, monkeypatch):
    """Rows, pages, holders and tokens as before: the requests can be submitted again."""
    from qwen3_engine_from_scratch_amd.engine import Engine, GenRequest

    monkeypatch.setattr(pc, "fork_pages_hip", lambda *args: None)  # the launch: bookkeeping only
    pool = _pool(blocks=12, rows=6)
    prefix = PagedKVCache(pool)
    prefix.reserve_slots(40)
    prefix.advance_seq_len(40)
    free, rows = sorted(pool.free_block_ids), sorted(pool._free_rows)
    reqs = [GenRequest(0, [1] * 5, 4, prefix=prefix), GenRequest(1, [1] * 20, 4),
            GenRequest(2, [2] * 9, 4, prefix=prefix, eos_token_id=7)]
    engine = _engine(pool, fail_at)
    engine._prefill_pieces = lambda r: Engine._prefill_pieces(engine, r)
    with pytest.raises(RuntimeError, match="a step"):
        Engine._prefill(engine, reqs)
    assert sorted(pool.free_block_ids) == free and sorted(pool._free_rows) == rows
    assert not pool._extra_holders and not prefix.freed and prefix.num_pages == 3
    assert all(r.cache is None and r.output_ids == [] and not r.eos_hit for r in reqs)
    engine._run_chunk = _engine(pool, 99)._run_chunk
    Engine._prefill(engine, reqs)
    assert [r.output_ids for r in reqs] == [[7], [7], [7]] and reqs[2].eos_hit


def test_too_few_rows_for_a_prefill_leave_nothing_behind():
    from qwen3_engine_from_scratch_amd.engine import Engine, GenRequest

    pool = _pool(blocks=12, rows=2)
    for prefill_chunk, n in ((8, 20), (None, 5)):  # in pieces, whole
        engine = _engine(pool, 99)
        engine.prefill_chunk, engine.device = prefill_chunk, torch.device("cpu")
        engine._prefill_pieces = lambda r: Engine._prefill_pieces(engine, r)
        engine._prefill_whole = lambda r: Engine._prefill_whole(engine, r)
        reqs = [GenRequest(i, [1] * n, 4) for i in range(3)]
        with pytest.raises(RuntimeError, match="rows exhausted"):
            Engine._prefill(engine, reqs)
        assert len(pool._free_rows) == 2 and all(r.cache is None for r in reqs)


def _fork_rows(k, v, table, seq_lens, src, dst, tokens, blocks):
    """The fork launch's part in the table, in blocks of 16."""
    for a, b, n, new in zip(src, dst, tokens, blocks):
        table[b] = -1
        table[b, :n // 16] = table[a, :n // 16]
        if n % 16:
            table[b, n // 16] = new
        seq_lens[b] = n


def _shared_and_full(monkeypatch, own_tail):
    """A handle of five (or three) pages, the first three shared, in a pool without a free
    block; and the page copies that are launched."""
    copies = []
    monkeypatch.setattr(pc, "fork_pages_hip", _fork_rows)
    monkeypatch.setattr(pc, "copy_pages_hip", lambda k, v, src, dst, tokens: copies.append((src, dst, tokens)))
    pool = _pool(blocks=5 if own_tail else 3)
    a = PagedKVCache(pool)
    a.reserve_slots(48)
    a.advance_seq_len(48)
    b = a.fork()
    if own_tail:
        b.reserve_slots(30)
        b.advance_seq_len(30)
    assert pool.free_count == 0
    return pool, a, b, copies


def test_truncate_in_a_full_pool_takes_a_page_it_gives_back(monkeypatch):
    pool, a, b, copies = _shared_and_full(monkeypatch, True)
    old, tail = list(b.block_table), b.block_table[3:]
    b.truncate(40)
    (src, dst, tokens), = copies
    assert src == [old[2]] and tokens == [8] and dst[0] in tail
    assert b.block_table == old[:2] + dst and b.num_pages == 3 and b.seq_len == 40
    assert pool.block_table_2d[b.row_id, :5].tolist() == b.block_table + [-1, -1]
    assert pool.free_block_ids == [x for x in tail if x not in dst]
    assert not pool.is_shared(old[2]) and pool.is_shared(old[1])
    a.free()
    b.free()
    assert sorted(pool.free_block_ids) == list(range(5)) and not pool._extra_holders


def test_truncate_without_a_page_to_copy_into_changes_nothing(monkeypatch):
    pool, a, b, copies = _shared_and_full(monkeypatch, False)
    before, pages = _state(pool), list(b.block_table)
    with pytest.raises(RuntimeError, match="OOM"):
        b.truncate(40)
    assert _state(pool) == before and b.block_table == pages and b.seq_len == 48 and not copies
    c = b.fork()  # a tail that others hold gives no page either
    c.truncate(16)
    before = _state(pool)
    with pytest.raises(RuntimeError, match="OOM"):
        b.truncate(10)
    assert _state(pool) == before and b.block_table == pages
