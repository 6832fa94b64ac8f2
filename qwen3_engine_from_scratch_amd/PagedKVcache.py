"""Paged KV cache: one shared physical block pool plus per-request handles.

Drop-in for qwen3/PagedKVcache.py of the reference engine.  Host-side
bookkeeping (free lists, row slots, page reservation, sequence lengths) keeps
the reference's semantics line for line in behaviour; the two device writes
go to HIP kernels:
  KVCachePool.update_kv_batch -> qwen3_kv_write_decode_bf16
  PagedKVCache.update         -> qwen3_kv_write_range_bf16
and the batched prefill write, which the reference runs as a per-request
loop of PagedKVCache.update (qwen3/attention.py:160-161), is one
slot-mapped launch (write_prefill_batch / qwen3_kv_write_slots_bf16).

Beyond the reference, requests can share pages (fork, fork_caches), give tokens back
(truncate) and have the pool's live pages moved together (KVCachePool.compact), on
the kernels of kernels/paged_cache.py.  One rule keeps every write path as it is:
the page that a request's next token falls into is never shared -- fork copies a
partly filled last page, truncate copies one that it leaves partly filled -- so only
whole, finished pages have several holders.  The pool counts them on the host.

Pool layout (num_blocks, num_layers, num_kv_heads, block_size, head_dim):
one (block, layer, head) chunk is block_size * head_dim contiguous bf16
(4 KiB at 16 x 128), the unit the decode kernel streams.
"""
from __future__ import annotations

import numpy as np
import torch

from . import _lib
from .kernels.paged_attention import update_kv_batch_hip
from .kernels.paged_cache import copy_pages_hip, fork_pages_hip, move_pages_hip

__all__ = ["KVCachePool", "PagedKVCache", "fork_caches", "shared_prefix_groups",
           "prefill_slot_mapping", "write_prefill_batch", "reserve_pages_bulk",
           "set_seq_lens_bulk", "PageIn"]


class KVCachePool:
    """Process-wide physical block pool shared by all requests
    (reference: qwen3/PagedKVcache.py:19-114)."""

    def __init__(self, num_blocks: int, num_layers: int, block_size: int,
                 num_kv_heads: int, head_dim: int, device=None, dtype=None,
                 max_seq_len: int = 2048, max_requests: int = 256):
        self.num_layers = num_layers
        self.block_size = block_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.max_seq_len = max_seq_len

        max_pages = (max_seq_len + block_size - 1) // block_size
        self.block_table_2d = torch.full(
            (max_requests, max_pages), -1, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(max_requests, dtype=torch.int32, device=device)
        self._free_rows = list(range(max_requests))
        self.max_requests = max_requests

        # Zero-initialised so never-written slots cannot hold NaN/inf.
        self.k_buffer = torch.zeros(num_blocks, num_layers, num_kv_heads,
                                    block_size, head_dim, device=device, dtype=dtype)
        self.v_buffer = torch.zeros(num_blocks, num_layers, num_kv_heads,
                                    block_size, head_dim, device=device, dtype=dtype)

        self.free_block_ids = list(range(num_blocks))
        self.total_blocks = num_blocks
        self._extra_holders = {}  # shared block -> its holders beyond the first

    def alloc(self, n: int):
        """Pops n block ids (LIFO from the tail) and zeroes their K/V, so a
        request never reads another request's stale tokens (:58-73)."""
        if len(self.free_block_ids) < n:
            raise RuntimeError(
                f"OOM: requested {n} blocks, {len(self.free_block_ids)} / {self.total_blocks} free")
        allocated = self.free_block_ids[-n:]
        del self.free_block_ids[-n:]
        if allocated:
            idx = torch.tensor(allocated, dtype=torch.long, device=self.k_buffer.device)
            self.k_buffer.index_fill_(0, idx, 0)
            self.v_buffer.index_fill_(0, idx, 0)
        return allocated

    def take_blocks(self, n: int) -> list:
        """Pops n block ids like alloc, without touching the device: the
        caller zeroes them (PageIn does, batched)."""
        if len(self.free_block_ids) < n:
            raise RuntimeError(
                f"OOM: requested {n} blocks, {len(self.free_block_ids)} / {self.total_blocks} free")
        allocated = self.free_block_ids[-n:]
        del self.free_block_ids[-n:]
        return allocated

    def free(self, block_ids: list):
        """Returns blocks; one that other requests still hold stays theirs."""
        if not self._extra_holders:
            self.free_block_ids.extend(block_ids)
            return
        for b in block_ids:
            left = self._extra_holders.get(b, 0)
            if left == 0:
                self.free_block_ids.append(b)
            elif left == 1:
                del self._extra_holders[b]
            else:
                self._extra_holders[b] = left - 1

    def share(self, block_ids: list):
        """One more holder for each of the blocks."""
        for b in block_ids:
            self._extra_holders[b] = self._extra_holders.get(b, 0) + 1

    def is_shared(self, block_id: int) -> bool:
        return block_id in self._extra_holders

    def compact(self, caches) -> int:
        """Moves the pages of the given handles into the lowest blocks (one launch per
        240 moves, the block table with them), so that what is free lies together at
        the pool's end; returns how many moved.  Blocks in use that these handles do
        not account for -- another handle's, a captured graph's own page -- stay where
        they are.  Tables change in place, so captured graphs stay valid; nothing may
        write into the pool on another stream meanwhile.  Blocks taken next come from
        the low end."""
        handles = list({id(c): c for c in caches}.values())
        holders: dict = {}
        for c in handles:
            if c._pool is not self:
                raise ValueError("a handle of another pool")
            for b in c.block_table:
                holders[b] = holders.get(b, 0) + 1
        used = self.total_blocks - len(self.free_block_ids)
        src = sorted(b for b, n in holders.items()
                     if b >= used and n == 1 + self._extra_holders.get(b, 0))
        dst = sorted(b for b in self.free_block_ids if b < used)[:len(src)]
        if src:
            move_pages_hip(self.k_buffer, self.v_buffer, self.block_table_2d, src, dst)
            to = dict(zip(src, dst))
            for c in handles:
                c.block_table = [to.get(b, b) for b in c.block_table]
            self._extra_holders = {to.get(b, b): n for b, n in self._extra_holders.items()}
            self.free_block_ids = list(set(self.free_block_ids).difference(dst).union(src))
        self.free_block_ids.sort(reverse=True)
        return len(src)

    @property
    def free_count(self):
        return len(self.free_block_ids)

    def alloc_row(self) -> int:
        """Reserves a resident-table row for a new request; its seq_len is
        reset to 0 (:85-93)."""
        if not self._free_rows:
            raise RuntimeError(
                f"OOM: request rows exhausted (max_requests={self.max_requests}); "
                "raise KVCachePool(max_requests=...)")
        row = self._free_rows.pop()
        self.seq_lens[row] = 0
        return row

    def free_row(self, row: int):
        self._free_rows.append(row)

    def update_kv_batch(self, layer_idx: int, k_new: torch.Tensor, v_new: torch.Tensor,
                        row_ids: torch.Tensor):
        """Decode write of one token per request (:99-114).

        k_new, v_new: (B, num_kv_heads, 1, head_dim); row_ids: (B,) int32.
        Pages must already be reserved (reserve_next) for this step.
        """
        update_kv_batch_hip(k_new.squeeze(2), v_new.squeeze(2), self.k_buffer, self.v_buffer,
                            self.seq_lens, self.block_table_2d, row_ids, layer_idx)


class PagedKVCache:
    """Per-request handle over the shared pool (reference:
    qwen3/PagedKVcache.py:117-228)."""

    freed = False  # its row is another request's by now

    def __init__(self, pool: KVCachePool):
        self._pool = pool
        self.seq_len = 0
        self.block_table = []
        self.row_id = pool.alloc_row()
        self.block_table_tensor = pool.block_table_2d[self.row_id]
        self.num_pages = 0

    def check_live(self):
        """Refuses a handle that was freed: what it would write into is another's."""
        if self.freed:
            raise ValueError("the handle was freed: its row may be another request's by now")

    def _allocate_block(self):
        self.check_live()
        max_pages = self.block_table_tensor.shape[0]
        assert self.num_pages < max_pages, \
            f"request exceeds max_seq_len ({self._pool.max_seq_len} tokens / {max_pages} pages)"
        new = self._pool.alloc(1)
        self.block_table.append(new[0])
        self.block_table_tensor[self.num_pages] = new[0]
        self.num_pages += 1

    def reserve_next(self):
        """Reserves the page the next decode token lands in (:152-162)."""
        self.check_live()
        need = (self.seq_len + 1 + self._pool.block_size - 1) // self._pool.block_size
        if need > self.num_pages:
            self._allocate_block()

    def get_kv(self, layer_idx: int):
        """All cached K, V of a layer as (1, Hkv, seq_len, D) (:164-175)."""
        if self.seq_len == 0 or not self.block_table:
            return None, None
        k_pages = [self._pool.k_buffer[pid, layer_idx] for pid in self.block_table]
        v_pages = [self._pool.v_buffer[pid, layer_idx] for pid in self.block_table]
        k = torch.cat(k_pages, dim=1)[:, :self.seq_len, :]
        v = torch.cat(v_pages, dim=1)[:, :self.seq_len, :]
        return k.unsqueeze(0), v.unsqueeze(0)

    def update(self, layer_idx: int, k_new: torch.Tensor, v_new: torch.Tensor):
        """Writes S_new tokens at positions seq_len .. seq_len+S_new-1 (:177-214).

        k_new, v_new: (B, num_kv_heads, S_new, head_dim); as in the reference
        only batch row 0 is written.  Pages are reserved first.
        """
        self.check_live()
        _, _, S_new, _ = k_new.shape
        pool = self._pool
        end_pos = self.seq_len + S_new
        need_blocks = (end_pos + pool.block_size - 1) // pool.block_size
        while len(self.block_table) < need_blocks:
            self._allocate_block()
        if S_new == 0:
            return
        assert 0 <= layer_idx < pool.num_layers
        k0 = k_new[0].transpose(0, 1)  # (S_new, Hkv, D) view
        v0 = v_new[0].transpose(0, 1)
        if k0.stride(2) != 1:
            k0 = k0.contiguous()
        if v0.stride(2) != 1:
            v0 = v0.contiguous()
        dev = _lib.require_hip(k0, v0, pool.k_buffer)
        lib = _lib.load()
        rc = lib.qwen3_kv_write_range_bf16(
            k0.data_ptr(), _lib.strides(k0, (0, 1)),
            v0.data_ptr(), _lib.strides(v0, (0, 1)),
            pool.k_buffer.data_ptr(), _lib.strides(pool.k_buffer, (0, 1, 2, 3)),
            pool.v_buffer.data_ptr(), _lib.strides(pool.v_buffer, (0, 1, 2, 3)),
            pool.k_buffer.shape[0], int(layer_idx), pool.k_buffer.shape[1],
            self.block_table_tensor.data_ptr(), self.num_pages,
            self.seq_len, S_new, pool.num_kv_heads, pool.head_dim, pool.block_size,
            _lib.stream_of(dev))
        _lib.check(rc, "qwen3_kv_write_range_bf16")

    def reserve_slots(self, n: int):
        """Reserves the pages of positions seq_len .. seq_len + n - 1 (as
        update does, :186-190) and returns their pool slots, block *
        block_size + offset, as an int64 numpy array."""
        self.check_live()
        bs = self._pool.block_size
        end = self.seq_len + n
        while len(self.block_table) < (end + bs - 1) // bs:
            self._allocate_block()
        p = np.arange(self.seq_len, end, dtype=np.int64)
        table = np.asarray(self.block_table, dtype=np.int64)
        return table[p // bs] * bs + p % bs

    def advance_seq_len(self, n: int = 1):
        self.check_live()
        self.seq_len += n
        self._pool.seq_lens[self.row_id] = self.seq_len

    def fork(self, tokens: int | None = None) -> "PagedKVCache":
        """A new handle that starts with this one's first `tokens` tokens (None: all):
        parallel samples of one prompt, requests behind a common prefix.  Whole pages
        are shared, a partly filled last one is copied; one launch."""
        return fork_caches([self], None if tokens is None else [tokens])[0]

    def truncate(self, tokens: int):
        """Gives back everything behind the first `tokens` tokens (draft tokens that
        were not accepted): pages that hold nothing of the rest are freed, and one
        that is left partly filled and has other holders is replaced by a copy (which
        takes a free block, or one of those that are given back)."""
        if self.freed or not 0 <= tokens <= self.seq_len:
            raise ValueError(f"cannot keep {tokens} of {self.seq_len} tokens")
        pool = self._pool
        bs = pool.block_size
        keep, rest = -(-tokens // bs), tokens % bs
        back = self.block_table[keep:]
        if rest and pool.is_shared(self.block_table[keep - 1]):
            old = self.block_table[keep - 1]
            own = [b for b in back if not pool.is_shared(b)]
            reuse = own and not pool.free_count  # in a full pool: one that is given back anyway
            new = own[0] if reuse else pool.take_blocks(1)[0]
            try:
                copy_pages_hip(pool.k_buffer, pool.v_buffer, [old], [new], [rest])
            except Exception:
                if not reuse:
                    pool.free([new])
                raise
            if reuse:
                back.remove(new)
            self.block_table[keep - 1] = new
            self.block_table_tensor[keep - 1] = new
            pool.free([old])
        if keep < self.num_pages:
            pool.free(back)
            del self.block_table[keep:]
            self.block_table_tensor[keep:self.num_pages] = -1
            self.num_pages = keep
        self.seq_len = tokens
        pool.seq_lens[self.row_id] = tokens

    def free(self):
        """Gives back the row and the pages; once: a second call finds nothing left."""
        if self.freed:
            return
        if self.block_table:
            self._pool.free(self.block_table)
            self.block_table = []
            self.num_pages = 0
        self.seq_len = 0
        self.freed = True
        self._pool.free_row(self.row_id)


def fork_caches(parents: list, tokens: list | None = None) -> list:
    """A new handle for every entry of `parents` (the same one may come several
    times), starting with its first tokens[i] tokens (None: all of them), in one
    launch: the block-table rows, the copies of the partly filled last pages and the
    lengths.  Takes a row a fork, and a block where the tokens end inside a page; a
    pool that has too few raises before anything changes."""
    if not parents:
        return []
    pool = parents[0]._pool
    bs = pool.block_size
    if tokens is None:
        tokens = [p.seq_len for p in parents]
    if len(tokens) != len(parents):
        raise ValueError(f"{len(tokens)} lengths for {len(parents)} forks")
    for p, n in zip(parents, tokens):
        if p._pool is not pool:
            raise ValueError("forks of several pools in one call")
        if p.freed:
            raise ValueError("a fork of a handle that was freed")
        if not 0 <= n <= p.seq_len:
            raise ValueError(f"cannot fork {n} of {p.seq_len} tokens")
    if len(pool._free_rows) < len(parents):
        raise RuntimeError(f"OOM: {len(parents)} request rows needed, {len(pool._free_rows)} free")
    ends_inside = [n % bs != 0 for n in tokens]
    need = sum(ends_inside)
    if pool.free_count < need:
        raise RuntimeError(
            f"OOM: requested {need} blocks, {pool.free_count} / {pool.total_blocks} free")
    rows = pool._free_rows[-len(parents):][::-1]
    fresh = iter(pool.free_block_ids[len(pool.free_block_ids) - need:])
    blocks = [next(fresh) if e else -1 for e in ends_inside]
    fork_pages_hip(pool.k_buffer, pool.v_buffer, pool.block_table_2d, pool.seq_lens,
                   [p.row_id for p in parents], rows, tokens, blocks)
    if need:
        pool.take_blocks(need)
    children = []
    for p, n, row, block in zip(parents, tokens, rows, blocks):
        c = PagedKVCache.__new__(PagedKVCache)
        c._pool = pool
        c.seq_len = n
        c.row_id = row  # its length is written by the launch
        pool._free_rows.pop()
        c.block_table_tensor = pool.block_table_2d[row]
        shared = p.block_table[:n // bs]
        pool.share(shared)
        c.block_table = shared if block < 0 else shared + [block]
        c.num_pages = len(c.block_table)
        children.append(c)
    return children


def shared_prefix_groups(caches: list) -> tuple[list, list, list]:
    """How a batch of handles shares its first pages, for
    paged_attention_decode_shared_hip: (order, cu_groups, shared_lens), host lists.
    order: a permutation of the handles that brings each group's together, what shares
    nothing last; group g is entries cu_groups[g] .. cu_groups[g + 1] - 1 of it, which hold
    their first shared_lens[g] tokens in the same (whole) pages.  Of nested prefixes (a
    system prompt, questions behind it) those are taken that save the most pages.  Valid
    as long as the handles only grow."""
    pool = caches[0]._pool if caches else None
    for c in caches:
        c.check_live()
        if c._pool is not pool:
            raise ValueError("handles of several pools in one batch")
    tables = [c.block_table for c in caches]
    order = sorted(range(len(caches)), key=lambda i: tables[i])

    def common(a, b):
        lo, hi = 0, min(len(a), len(b))
        while lo < hi:  # the first lo pages are common, more than hi are not
            mid = (lo + hi + 1) // 2
            if a[lo:mid] == b[lo:mid]:
                lo = mid
            else:
                hi = mid - 1
        return lo

    # The sorted handles' common prefixes form a tree: a node is a range of them and the
    # pages that all of it begins with.  Bottom up, a node makes a group of the handles that
    # have none below it and of those groups that save no more by themselves.
    #   open node: pages, first handle, handles without a group, groups (handles, pages)
    stack = [(0, 0, [], [])]
    for i in range(1, len(order) + 1):
        pages = common(tables[order[i - 1]], tables[order[i]]) if i < len(order) else 0
        lo, free, groups = i - 1, order[i - 1:i], []
        while pages < stack[-1][0]:
            n, lo, more_free, more_groups = stack.pop()
            free, groups = more_free + free, more_groups + groups
            keep = [g for g in groups if (len(g[0]) - 1) * g[1] > len(g[0]) * n]
            lost = sum((len(g[0]) - 1) * g[1] for g in groups) \
                - sum((len(g[0]) - 1) * g[1] for g in keep)
            joined = free + [h for g in groups if g not in keep for h in g[0]]
            if (len(joined) - 1) * n > lost:
                free, groups = [], keep + [(joined, n)]
        if pages > stack[-1][0]:
            stack.append((pages, lo, free, groups))
        else:
            top = stack.pop()
            stack.append((*top[:2], top[2] + free, top[3] + groups))
    groups = stack[0][3]  # below the root, which shares nothing
    grouped = [i for members, _ in groups for i in members]
    alone = sorted(set(order).difference(grouped))
    cu = [0]
    for members, _ in groups:
        cu.append(cu[-1] + len(members))
    bs = pool.block_size if pool is not None else 0
    return grouped + alone, cu, [pages * bs for _, pages in groups]


class PageIn:
    """Batched page reservation with no host synchronisation: new blocks are
    taken on the host, and their table entries plus the zeroing of their K/V
    go to the device as one asynchronous copy from pinned memory and one
    launch (qwen3_page_in_bf16).  Two pinned staging buffers alternate, so a
    buffer is rewritten only after the copy of the call before the previous
    one has run (the caller synchronises once per step, as the engine does)."""

    def __init__(self, pool: KVCachePool, capacity: int):
        assert pool.k_buffer.is_contiguous() and pool.v_buffer.is_contiguous()
        self.pool = pool
        self.cap = capacity
        self._host = [torch.empty(3 * capacity, dtype=torch.int32, pin_memory=True)
                      for _ in range(2)]
        self._dev = torch.empty(3 * capacity, dtype=torch.int32, device=pool.k_buffer.device)
        self._flip = 0

    def reserve(self, caches, tokens) -> int:
        """Gives every handle enough pages for tokens[i] tokens; returns the
        number of blocks mapped."""
        pool = self.pool
        bs = pool.block_size
        max_pages = pool.block_table_2d.shape[1]
        want = []
        for c, n in zip(caches, tokens):
            c.check_live()
            k = (int(n) + bs - 1) // bs - c.num_pages
            if k > 0:
                assert c.num_pages + k <= max_pages, \
                    f"request exceeds max_seq_len ({pool.max_seq_len} tokens / {max_pages} pages)"
                want.append((c, k))
        total = sum(k for _, k in want)
        if total == 0:
            return 0
        assert total <= self.cap, f"{total} new pages in one step (staging holds {self.cap})"
        ids = pool.take_blocks(total)
        h = self._host[self._flip]
        self._flip ^= 1
        # rows | page columns | block ids, filled through a numpy view of the
        # pinned buffer (element-wise tensor writes cost microseconds each)
        hn = h.numpy()
        counts = [k for _, k in want]
        hn[:total] = np.repeat([c.row_id for c, _ in want], counts)
        hn[total:2 * total] = np.concatenate(
            [np.arange(c.num_pages, c.num_pages + k) for c, k in want])
        hn[2 * total:3 * total] = ids
        i = 0
        for c, k in want:
            c.block_table.extend(ids[i:i + k])
            c.num_pages += k
            i += k
        d = self._dev[:3 * total]
        d.copy_(h[:3 * total], non_blocking=True)
        bt = pool.block_table_2d
        kb = pool.k_buffer
        rc = _lib.load().qwen3_page_in_bf16(
            bt.data_ptr(), bt.stride(0), bt.shape[0], bt.shape[1], d.data_ptr(), total,
            kb.data_ptr(), pool.v_buffer.data_ptr(), kb[0].numel(), kb.shape[0],
            _lib.stream_of(kb.device))
        _lib.check(rc, "qwen3_page_in_bf16")
        return total


def reserve_pages_bulk(caches, tokens: list) -> None:
    """Gives every handle enough pages for tokens[i] tokens with one pool
    allocation (one zeroing launch) and one block-table write for the whole
    batch, instead of a device write per page (_allocate_block).  Used by the
    batching engine once per step."""
    pool = caches[0]._pool
    bs = pool.block_size
    max_pages = pool.block_table_2d.shape[1]
    want = []
    for c, n in zip(caches, tokens):
        c.check_live()
        k = (int(n) + bs - 1) // bs - c.num_pages
        if k > 0:
            assert c.num_pages + k <= max_pages, \
                f"request exceeds max_seq_len ({pool.max_seq_len} tokens / {max_pages} pages)"
            want.append((c, k))
    total = sum(k for _, k in want)
    if total == 0:
        return
    ids = pool.alloc(total)
    rows, cols, vals = [], [], []
    for c, k in want:
        new, ids = ids[:k], ids[k:]
        rows += [c.row_id] * k
        cols += range(c.num_pages, c.num_pages + k)
        vals += new
        c.block_table.extend(new)
        c.num_pages += k
    idx = torch.tensor([rows, cols, vals], dtype=torch.int64).to(pool.block_table_2d.device)
    pool.block_table_2d.index_put_((idx[0], idx[1]), idx[2].to(torch.int32))


def set_seq_lens_bulk(caches) -> None:
    """Writes every handle's host seq_len into the resident seq_lens table
    with one copy (the batched form of advance_seq_len's device write)."""
    pool = caches[0]._pool
    for c in caches:
        c.check_live()
    idx = torch.tensor([[c.row_id for c in caches], [c.seq_len for c in caches]],
                       dtype=torch.int64).to(pool.seq_lens.device)
    pool.seq_lens.index_put_((idx[0],), idx[1].to(torch.int32))


def prefill_slot_mapping(caches, S: int, device) -> torch.Tensor:
    """Slot of every (request, padded position) of a right-padded prefill
    batch: the reference's per-request update writes all S positions from
    each request's seq_len (pads included, qwen3/attention.py:160-161), so the
    mapping covers them too.  Reserves the pages the same way."""
    bs = caches[0]._pool.block_size
    slots = np.empty((len(caches), S), dtype=np.int64)
    pos = np.arange(S, dtype=np.int64)
    for i, c in enumerate(caches):
        c.check_live()
        end_pos = c.seq_len + S
        need = (end_pos + bs - 1) // bs
        while len(c.block_table) < need:
            c._allocate_block()
        p = c.seq_len + pos
        table = np.asarray(c.block_table, dtype=np.int64)
        slots[i] = table[p // bs] * bs + p % bs
    return torch.from_numpy(slots.reshape(-1)).to(device, non_blocking=False)


def write_prefill_batch(caches, layer_idx: int, k: torch.Tensor, v: torch.Tensor,
                        slot_mapping: torch.Tensor | None = None):
    """One-launch equivalent of `for i, c in enumerate(caches): c.update(layer_idx,
    k[i:i+1], v[i:i+1])` (qwen3/attention.py:160-161).

    k, v: (B, Hkv, S, D).  `slot_mapping` (B*S,) int64 from prefill_slot_mapping
    can be built once per step and shared by every layer.
    """
    B, Hkv, S, D = k.shape
    pool = caches[0]._pool
    if slot_mapping is None:
        slot_mapping = prefill_slot_mapping(caches, S, k.device)
    assert slot_mapping.dtype == torch.int64 and slot_mapping.numel() == B * S
    assert 0 <= layer_idx < pool.num_layers
    # (B, Hkv, S, D) -> token-major (B*S, Hkv, D) view when strides allow.
    kt = k.transpose(1, 2).reshape(B * S, Hkv, D)
    vt = v.transpose(1, 2).reshape(B * S, Hkv, D)
    dev = _lib.require_hip(kt, vt, pool.k_buffer, slot_mapping)
    lib = _lib.load()
    rc = lib.qwen3_kv_write_slots_bf16(
        kt.data_ptr(), _lib.strides(kt, (0, 1)),
        vt.data_ptr(), _lib.strides(vt, (0, 1)),
        pool.k_buffer.data_ptr(), _lib.strides(pool.k_buffer, (0, 1, 2, 3)),
        pool.v_buffer.data_ptr(), _lib.strides(pool.v_buffer, (0, 1, 2, 3)),
        pool.k_buffer.shape[0], int(layer_idx), pool.k_buffer.shape[1],
        slot_mapping.contiguous().data_ptr(), B * S,
        Hkv, D, pool.block_size, _lib.stream_of(dev))
    _lib.check(rc, "qwen3_kv_write_slots_bf16")
