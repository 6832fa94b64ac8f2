"""Oracle for the attention of a chunk of new tokens over a paged cache.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py).  The definition in 64 bits, one
token and one head at a time over the keys gathered through the block table; the
reference engine has no counterpart.  Pinned by the decode oracle (chunks of one
token) and by the varlen closed form (nothing cached).
"""
from __future__ import annotations

import torch


def keys_of_row(table_row, reach: int, block_size: int, num_blocks: int):
    """(pages, slots) of the positions 0 .. reach - 1 that may be attended: those a
    row of the table addresses, in blocks of the pool; and their positions."""
    pos = torch.arange(max(0, min(reach, len(table_row) * block_size)))
    page = torch.as_tensor(table_row).long()[pos // block_size]
    ok = (page >= 0) & (page < num_blocks)
    return page[ok], (pos % block_size)[ok], pos[ok]


def paged_chunk_ref(q, k_layer, v_layer, table, seq_lens, row_ids, cu, block_size, scale):
    """q (T, Hq, D); k_layer, v_layer (blocks, Hkv, block_size, D); table (rows, pages),
    seq_lens (rows,), row_ids (B,), cu (B + 1,) on the CPU.  Returns (out, spread): out
    (T, Hq, D) float64, NaN where no sequence has the row; spread = sum_j p_ij |v_j|, by
    which a rounding of P is bounded.  Runs where q lies."""
    T, hq, D = q.shape
    hkv = k_layer.shape[1]
    G = hq // hkv
    out = torch.full((T, hq, D), float("nan"), dtype=torch.float64, device=q.device)
    spread = torch.zeros_like(out)
    for b in range(len(cu) - 1):
        s0, s1 = int(cu[b]), int(cu[b + 1])
        n = s1 - s0
        if n <= 0:
            continue
        row = int(row_ids[b])
        out[s0:s1] = 0
        if row < 0 or row >= table.shape[0]:
            continue
        ctx = int(seq_lens[row])
        page, slot, pos = (x.to(q.device) for x in keys_of_row(
            table[row].tolist(), ctx + n, block_size, k_layer.shape[0]))
        if not len(pos):
            continue
        kc, vc = (x[page, :, slot].double().permute(1, 0, 2) for x in (k_layer, v_layer))
        for i0 in range(0, n, 256):  # rows at a time: the scores of a long context in 64 bits
            i1 = min(n, i0 + 256)
            qs = q[s0 + i0:s0 + i1].double().view(i1 - i0, hkv, G, D).permute(1, 0, 2, 3)
            x = torch.matmul(qs.reshape(hkv, (i1 - i0) * G, D),
                             kc.transpose(1, 2).contiguous()) * scale
            last = ctx + torch.arange(i0, i1, device=q.device).repeat_interleave(G)
            x = x.masked_fill(pos[None, :] > last[:, None], float("-inf"))
            m = x.amax(-1, keepdim=True)
            p = torch.exp(x - torch.where(m == float("-inf"), 0.0, m))
            l = p.sum(-1, keepdim=True)
            w = torch.where(l > 0, p / torch.where(l > 0, l, 1.0), 0.0)
            for dst, val in ((out, vc), (spread, vc.abs())):
                y = torch.matmul(w, val.contiguous()).view(hkv, i1 - i0, G, D)
                dst[s0 + i0:s0 + i1] = y.permute(1, 0, 2, 3).reshape(i1 - i0, hq, D)
    return out, spread
