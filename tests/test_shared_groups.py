"""shared_prefix_groups: the groups that save the most pages, on handles of many shapes (CPU)."""
import random
from types import SimpleNamespace

import pytest
import torch

from qwen3_engine_from_scratch_amd.PagedKVcache import (KVCachePool, PagedKVCache,
                                                        shared_prefix_groups)


class Handle:
    def __init__(self, table, pool):
        self.block_table, self._pool = table, pool

    def check_live(self):
        pass


def common(a, b):
    n = 0
    while n < min(len(a), len(b)) and a[n] == b[n]:
        n += 1
    return n


def most_saved(tables):
    """The best division of the tables into groups, by trying all."""
    def best(left):
        if not left:
            return 0
        most = 0
        for k in range(1 << (len(left) - 1)):  # who is with the first one
            group = [left[0]] + [t for i, t in enumerate(left[1:]) if k >> i & 1]
            pages = min((common(group[0], t) for t in group[1:]), default=0)
            most = max(most, pages * (len(group) - 1)
                       + best([t for i, t in enumerate(left[1:]) if not k >> i & 1]))
        return most

    return best(tables)


def test_groups_save_the_most_pages():
    rnd = random.Random(1)
    pool = SimpleNamespace(block_size=16)
    for _ in range(400):
        fresh, tables = 100, []
        for _ in range(rnd.randint(0, 7)):
            t = []
            if tables and rnd.random() < 0.8:
                b = rnd.choice(tables)
                t = b[:rnd.randint(0, len(b))]
            own = rnd.randint(0, 4)
            tables.append(t + list(range(fresh, fresh + own)))
            fresh += own
        order, cu, shared = shared_prefix_groups([Handle(t, pool) for t in tables])
        assert sorted(order) == list(range(len(tables))) and cu[0] == 0 and len(cu) == len(shared) + 1
        saved = 0
        for g, tokens in enumerate(shared):
            members = [tables[i] for i in order[cu[g]:cu[g + 1]]]
            pages = tokens // 16
            assert len(members) > 1 and tokens > 0 and tokens % 16 == 0
            assert all(m[:pages] == members[0][:pages] and len(m) >= pages for m in members)
            saved += (len(members) - 1) * pages
        assert saved == most_saved(tables), tables
        rest = order[cu[-1]:]
        assert rest == sorted(rest)


def test_long_chains_and_large_groups():
    pool = SimpleNamespace(block_size=32)
    chain = [Handle(list(range(i)), pool) for i in range(1200)]  # each behind the one before
    order, cu, shared = shared_prefix_groups(chain)
    assert sorted(order) == list(range(1200)) and cu[-1] <= 1200
    big = [Handle(list(range(3000)) + [5000 + i], pool) for i in range(256)]
    assert shared_prefix_groups(big)[1:] == ([0, 256], [96000])


def test_what_is_refused():
    pools = [KVCachePool(4, 1, 16, 1, 128, device="cpu", dtype=torch.bfloat16, max_seq_len=64,
                         max_requests=4) for _ in range(2)]
    a, b = PagedKVCache(pools[0]), PagedKVCache(pools[1])
    with pytest.raises(ValueError, match="several pools"):
        shared_prefix_groups([a, b])
    a.free()
    with pytest.raises(ValueError, match="freed"):
        shared_prefix_groups([a])
    assert shared_prefix_groups([]) == ([], [0], [])
