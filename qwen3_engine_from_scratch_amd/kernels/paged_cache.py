"""Pages of the KV pool copied, forked and moved on the gfx950 HIP kernels
(include/qwen3_model_ops.h).

No counterpart in the reference engine, whose requests never share a page.  The
plans are host lists (the pool's bookkeeping is on the host); they travel in the
launch, so a call neither synchronises nor waits for a staging copy, and the
checks (every id in range, no block written twice or read and written) are done
before anything is launched.  KVCachePool and PagedKVCache call these for fork,
truncate and compact.
"""
from __future__ import annotations

from array import array

import torch

from .. import _lib

__all__ = ["copy_pages_hip", "fork_pages_hip", "move_pages_hip"]


def _list(values, n: int, what: str) -> array:
    """A host list as 32-bit integers."""
    try:
        a = array("i", values)
    except OverflowError:
        raise ValueError(f"{what} does not fit 32 bits") from None
    if len(a) != n:
        raise ValueError(f"{what} has {len(a)} entries, expected {n}")
    return a


def _at(a: array) -> int:
    return a.buffer_info()[0]


def _pool(k_buffer, v_buffer):
    """The pool as the C entries take it: its blocks must be contiguous chunks."""
    assert k_buffer.dim() == 5 and v_buffer.shape == k_buffer.shape, \
        "the pool is (num_blocks, num_layers, num_kv_heads, block_size, head_dim)"
    assert k_buffer.dtype == torch.bfloat16 and v_buffer.dtype == torch.bfloat16, \
        "HIP page kernels are bf16 only"
    assert k_buffer.is_contiguous() and v_buffer.is_contiguous(), "the pool must be contiguous"
    n, layers, heads, bs, d = k_buffer.shape
    return (k_buffer.data_ptr(), v_buffer.data_ptr(), layers * heads * bs * d, d, bs, n)


def _table(block_table_2d):
    assert block_table_2d.dtype == torch.int32 and block_table_2d.dim() == 2 \
        and block_table_2d.stride(1) == 1, "block_table_2d rows must be contiguous int32"
    return (block_table_2d.data_ptr(), block_table_2d.stride(0), *block_table_2d.shape)


def copy_pages_hip(k_buffer: torch.Tensor, v_buffer: torch.Tensor, src, dst, tokens=None) -> None:
    """Block dst[i] becomes a copy of block src[i], all layers, K and V: its first
    tokens[i] slots, the others zero (None: whole blocks).  src, dst, tokens: host
    lists.  No block may be written twice, or read and written."""
    n = len(src)
    pool = _pool(k_buffer, v_buffer)
    s, d = _list(src, n, "src"), _list(dst, n, "dst")
    t = None if tokens is None else _list(tokens, n, "tokens")
    dev = _lib.require_hip(k_buffer, v_buffer)
    with _lib.on_device(dev):
        rc = _lib.load().qwen3_page_copy_bf16(
            *pool, _at(s), _at(d), None if t is None else _at(t), n, _lib.stream_of(dev))
    _lib.check(rc, "qwen3_page_copy_bf16")


def fork_pages_hip(k_buffer: torch.Tensor, v_buffer: torch.Tensor, block_table_2d: torch.Tensor,
                   seq_lens: torch.Tensor, src_rows, dst_rows, tokens, new_blocks) -> None:
    """Row dst_rows[i] takes over the pages of the first tokens[i] tokens of row
    src_rows[i]: whole pages are shared, a partly filled last one is copied into block
    new_blocks[i] (its other slots zero; the block is not used where the tokens fill
    whole pages, -1 will do).  The row's other entries become -1 and
    seq_lens[dst_rows[i]] = tokens[i].  Host lists; who else holds a shared page is
    the caller's bookkeeping (PagedKVCache.fork keeps it)."""
    n = len(src_rows)
    pool, table = _pool(k_buffer, v_buffer), _table(block_table_2d)
    assert seq_lens.dtype == torch.int32 and seq_lens.is_contiguous() \
        and seq_lens.numel() >= block_table_2d.shape[0]
    lists = (_list(src_rows, n, "src_rows"), _list(dst_rows, n, "dst_rows"),
             _list(tokens, n, "tokens"), _list(new_blocks, n, "new_blocks"))
    dev = _lib.require_hip(k_buffer, v_buffer, block_table_2d, seq_lens)
    with _lib.on_device(dev):
        rc = _lib.load().qwen3_page_fork_bf16(*pool, *table, seq_lens.data_ptr(),
                                              *map(_at, lists), n, _lib.stream_of(dev))
    _lib.check(rc, "qwen3_page_fork_bf16")


def move_pages_hip(k_buffer: torch.Tensor, v_buffer: torch.Tensor, block_table_2d: torch.Tensor,
                   src, dst) -> None:
    """Block src[i] moves to block dst[i] (host lists): K and V of all layers are
    copied, and every entry of the table that names src[i] names dst[i] afterwards.  No
    block may be named twice."""
    n = len(src)
    pool, table = _pool(k_buffer, v_buffer), _table(block_table_2d)
    s, d = _list(src, n, "src"), _list(dst, n, "dst")
    dev = _lib.require_hip(k_buffer, v_buffer, block_table_2d)
    with _lib.on_device(dev):
        rc = _lib.load().qwen3_page_move_bf16(*pool, *table, _at(s), _at(d), n,
                                              _lib.stream_of(dev))
    _lib.check(rc, "qwen3_page_move_bf16")
