"""Shared-prefix decode attention refuses bad calls before anything is launched (CPU)."""
import ctypes

import pytest
import torch

from qwen3_engine_from_scratch_amd import _lib

FAKE = 1 << 20  # 16-byte aligned, never dereferenced on these paths


def _s(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _call(**over):
    a = dict(q=FAKE, qs=_s(4096, 128), k=FAKE, ks=_s(65536, 2048, 128), v=FAKE,
             vs=_s(65536, 2048, 128), nb=64, bt=FAKE, bts=8, rows=4, mp=8, sl=FAKE, bias=1, rid=None,
             cu=FAKE, sh=FAKE, ng=1, out=FAKE, os=_s(4096, 128), B=2, H=32, Hk=8, D=128, bs=16,
             scale=0.088, ws=FAKE, wsb=1 << 40, stream=None)
    a.update(over)
    return _lib.load().qwen3_paged_decode_shared_bf16(
        a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["nb"], a["bt"], a["bts"], a["rows"],
        a["mp"], a["sl"], a["bias"], a["rid"], a["cu"], a["sh"], a["ng"], a["out"], a["os"], a["B"],
        a["H"], a["Hk"], a["D"], a["bs"], a["scale"], a["ws"], a["wsb"], a["stream"])


@pytest.mark.parametrize("code,over", [
    (-3, dict(D=64)), (-3, dict(bs=8)), (-3, dict(bs=24)), (-3, dict(H=30)), (-3, dict(H=8 * 17)),
    (-3, dict(Hk=0)), (-3, dict(ks=_s(65536, 2048, 64))), (-3, dict(vs=_s(65536, 2048, 1 << 25))),
    (-3, dict(B=1025)), (-1, dict(q=None)), (-1, dict(k=None)), (-1, dict(v=None)),
    (-1, dict(bt=None)), (-1, dict(sl=None)), (-1, dict(cu=None)), (-1, dict(sh=None)),
    (-1, dict(out=None)), (-1, dict(qs=None)), (-1, dict(os=None)), (-1, dict(bts=4)),
    (-1, dict(nb=0)), (-1, dict(rows=0)), (-1, dict(mp=0)), (-1, dict(B=-1)), (-1, dict(ng=-1)),
    (-1, dict(ng=3)), (-1, dict(scale=0.0)), (-1, dict(scale=-1.0)), (-1, dict(scale=float("nan"))),
    (-1, dict(scale=float("inf"))), (-1, dict(mp=1 << 27, bts=1 << 27)),
    (-1, dict(B=1000, mp=1 << 21, bts=1 << 21)),
    (-2, dict(q=FAKE + 2)), (-2, dict(out=FAKE + 8)), (-2, dict(qs=_s(4097, 128))),
    (-2, dict(ks=_s(65536, 2048, 132))), (-4, dict(ws=None)), (-4, dict(wsb=8)),
    (-2, dict(ws=FAKE + 4)),
])
def test_refuses(code, over):
    assert _call(**over) == code, _lib.load().qwen3_attn_last_error()


def test_nothing_to_do_is_no_error():
    assert _call(B=0, ng=0) == 0


def test_workspace_bytes():
    f = _lib.load().qwen3_paged_decode_shared_workspace_bytes
    assert f(2, 32, 8, 128) > 0 and f(1024, 64, 8, 128) > f(2, 64, 8, 128)
    for bad in ((0, 32, 8, 128), (1025, 32, 8, 128), (2, 30, 8, 128), (2, 32, 8, 64), (2, 34, 2, 128)):
        assert f(*bad) == 0


def test_wrapper_refuses():
    from qwen3_engine_from_scratch_amd.kernels.paged_attention import paged_attention_decode_shared_hip

    def call(**over):
        t = dict(q=torch.zeros(4, 16, 128, dtype=torch.bfloat16),
                 k=torch.zeros(3, 8, 16, 128, dtype=torch.bfloat16),
                 v=torch.zeros(3, 8, 16, 128, dtype=torch.bfloat16),
                 bt=torch.zeros(4, 2, dtype=torch.int32), sl=torch.zeros(4, dtype=torch.int32),
                 rows=torch.zeros(4, dtype=torch.int32), cu=torch.tensor([0, 4], dtype=torch.int32),
                 sh=torch.tensor([16], dtype=torch.int32), bs=16)
        t.update(over)
        return paged_attention_decode_shared_hip(t["q"], t["k"], t["v"], t["bt"], t["sl"], t["rows"],
                                                 t["cu"], t["sh"], t["bs"])

    with pytest.raises(RuntimeError, match="no CPU fallback"):
        call()
    for over in (dict(q=torch.zeros(4, 16, 128)), dict(bs=32), dict(k=torch.zeros(3, 8, 16, 128)),
                 dict(cu=torch.tensor([0, 4])), dict(sh=torch.tensor([16])),
                 dict(sh=torch.zeros(2, dtype=torch.int32)), dict(bt=torch.zeros(4, 2)),
                 dict(cu=torch.zeros(6, dtype=torch.int32), sh=torch.zeros(5, dtype=torch.int32)),
                 dict(rows=torch.zeros(3, dtype=torch.int32)),
                 dict(rows=None, bt=torch.zeros(3, 2, dtype=torch.int32)),
                 dict(sl=torch.zeros(1, dtype=torch.int32)),
                 dict(v=torch.zeros(3, 4, 16, 128, dtype=torch.bfloat16))):
        with pytest.raises(AssertionError):
            call(**over)
