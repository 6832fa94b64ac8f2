"""Chunk attention's oracle is pinned, and its entry points refuse bad calls before
anything is launched (CPU)."""
import ctypes

import pytest
import torch

from oracle import decode as od
from oracle import inputs as oi
from oracle import prefill as op
from oracle.chunk import paged_chunk_ref
from qwen3_engine_from_scratch_amd import _lib

FAKE = 1 << 20  # 16-byte aligned, never dereferenced on these paths


def _s(*v):
    return (ctypes.c_int64 * len(v))(*v)


def test_chunks_of_one_token_are_decode():
    case = oi.make_decode_case([37, 1, 200], 16, 8, 128, 16, seed=1)
    B = len(case.seq_lens)
    out, _ = paged_chunk_ref(case.q, case.k_pool, case.v_pool, case.block_table, case.seq_lens,
                             case.row_ids, torch.arange(B + 1), 16, 128 ** -0.5)
    ref = od.dense_decode_ref(case.q, case.k_pool, case.v_pool, case.block_table, case.seq_lens,
                              case.row_ids, 16)
    assert (out - ref).abs().max() < 1e-9


def test_chunks_with_nothing_cached_are_prefill():
    c = oi.make_prefill_case([40, 16, 1], 16, 8, 128, seed=2)
    lens, bs = [40, 16, 1], 16
    pages = [-(-n // bs) for n in lens]
    table = torch.full((3, max(pages)), -1)
    k = torch.zeros(sum(pages), 8, bs, 128, dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    at = 0
    for b, n in enumerate(lens):
        table[b, :pages[b]] = torch.arange(at, at + pages[b])
        s = int(c.cu_seqlens[b])
        for i in range(n):
            k[at + i // bs, :, i % bs] = c.k[s + i]
            v[at + i // bs, :, i % bs] = c.v[s + i]
        at += pages[b]
    out, spread = paged_chunk_ref(c.q, k, v, table, torch.zeros(3), torch.arange(3), c.cu_seqlens,
                                  bs, c.scale)
    ref = op.varlen_attention_ref(c.q, c.k, c.v, c.cu_seqlens, c.scale, dtype=torch.float64)
    assert (out - ref).abs().max() < 1e-9 and (spread >= out.abs() - 1e-12).all()


def _call(**over):
    a = dict(q=FAKE, qs=_s(4096, 128), k=FAKE, ks=_s(65536, 2048, 128), v=FAKE,
             vs=_s(65536, 2048, 128), nb=64, bt=FAKE, bts=8, rows=4, mp=8, sl=FAKE, rid=None,
             cu=FAKE, out=FAKE, os=_s(4096, 128), B=2, mc=5, T=10, H=32, Hk=8, D=128, bs=16,
             scale=0.088, ws=FAKE, wsb=1 << 40, stream=None)
    a.update(over)
    return _lib.load().qwen3_paged_chunk_bf16(
        a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["nb"], a["bt"], a["bts"], a["rows"],
        a["mp"], a["sl"], a["rid"], a["cu"], a["out"], a["os"], a["B"], a["mc"], a["T"], a["H"],
        a["Hk"], a["D"], a["bs"], a["scale"], a["ws"], a["wsb"], a["stream"])


@pytest.mark.parametrize("code,over", [
    (-3, dict(D=64)), (-3, dict(bs=8)), (-3, dict(bs=24)), (-3, dict(H=30)), (-3, dict(H=8 * 17)),
    (-3, dict(Hk=0)), (-3, dict(ks=_s(65536, 2048, 64))), (-3, dict(vs=_s(65536, 2048, 1 << 25))),
    (-1, dict(q=None)), (-1, dict(k=None)), (-1, dict(v=None)), (-1, dict(bt=None)),
    (-1, dict(sl=None)), (-1, dict(cu=None)), (-1, dict(out=None)), (-1, dict(qs=None)),
    (-1, dict(os=None)), (-1, dict(bts=4)), (-1, dict(nb=0)), (-1, dict(rows=0)),
    (-1, dict(mp=0)), (-1, dict(B=-1)), (-1, dict(mc=-1)), (-1, dict(T=-1)),
    (-1, dict(T=1 << 31)), (-1, dict(T=(1 << 31) - 1)), (-1, dict(scale=0.0)),
    (-1, dict(scale=-1.0)), (-1, dict(scale=float("nan"))), (-1, dict(scale=float("inf"))),
    (-1, dict(mp=1 << 27, bts=1 << 27)),
    (-2, dict(q=FAKE + 2)), (-2, dict(out=FAKE + 8)), (-2, dict(qs=_s(4097, 128))),
    (-2, dict(ks=_s(65536, 2048, 132))), (-4, dict(ws=None)), (-4, dict(wsb=8)),
    (-2, dict(ws=FAKE + 4)),
])
def test_chunk_refuses(code, over):
    assert _call(**over) == code, _lib.load().qwen3_attn_last_error()


def test_nothing_to_do_is_no_error():
    for over in (dict(B=0), dict(mc=0), dict(T=0)):
        assert _call(**over) == 0


def test_workspace_bytes():
    f = _lib.load().qwen3_paged_chunk_workspace_bytes
    assert f(2, 5, 10, 32, 8, 128) > 0
    for bad in ((0, 5, 10, 32, 8, 128), (2, 0, 10, 32, 8, 128), (2, 5, 0, 32, 8, 128),
                (2, 5, 10, 30, 8, 128), (2, 5, 10, 32, 8, 64), (2, 5, 10, 34, 2, 128)):
        assert f(*bad) == 0


def test_wrapper_refuses():
    from qwen3_engine_from_scratch_amd.kernels.paged_attention import paged_attention_chunk_hip

    def call(**over):
        t = dict(q=torch.zeros(4, 16, 128, dtype=torch.bfloat16),
                 k=torch.zeros(3, 8, 16, 128, dtype=torch.bfloat16),
                 v=torch.zeros(3, 8, 16, 128, dtype=torch.bfloat16),
                 bt=torch.zeros(2, 2, dtype=torch.int32), sl=torch.zeros(2, dtype=torch.int32),
                 rows=torch.zeros(2, dtype=torch.int32), cu=torch.tensor([0, 2, 4], dtype=torch.int32),
                 bs=16)
        t.update(over)
        return paged_attention_chunk_hip(t["q"], t["k"], t["v"], t["bt"], t["sl"], t["rows"],
                                         t["cu"], t["bs"], max_chunk=2)

    with pytest.raises(RuntimeError, match="no CPU fallback"):
        call()
    for over in (dict(q=torch.zeros(4, 16, 128)), dict(bs=32), dict(k=torch.zeros(3, 8, 16, 128)),
                 dict(cu=torch.tensor([0, 2, 4])), dict(bt=torch.zeros(2, 2)),
                 dict(rows=torch.zeros(3, dtype=torch.int32)),
                 dict(rows=None, cu=torch.tensor([0, 1, 2, 3], dtype=torch.int32)),
                 dict(sl=torch.zeros(1, dtype=torch.int32)),
                 dict(v=torch.zeros(3, 4, 16, 128, dtype=torch.bfloat16))):
        with pytest.raises(AssertionError):
            call(**over)


def test_a_grid_beyond_32_bits_is_refused():
    assert _call(B=100000, mc=1 << 20, T=1 << 20, rows=100000) == -1
    assert b"grid too large" in _lib.load().qwen3_attn_last_error()
