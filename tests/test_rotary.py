"""Rotary frequencies against their laws and the transformers library's, refusals of
the entry points (CPU)."""
import ctypes
import math

import pytest
import torch

from qwen3_engine_from_scratch_amd import _lib
from qwen3_engine_from_scratch_amd.kernels.rotary import (Rotary, make_rotary,
                                                          rotary_embedding_decode_hip,
                                                          rotary_embedding_hip,
                                                          rotary_embedding_prefill_hip,
                                                          rotary_frequencies)

FAKE = 1 << 20
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}


def test_default_and_linear():
    f, m = rotary_frequencies(128, 1e6)
    assert m == 1.0 and f.dtype == torch.float64 and f.shape == (64,)
    for i in (0, 1, 31, 63):
        assert math.isclose(float(f[i]), 1e6 ** (-2 * i / 128), rel_tol=1e-13)
    g, m = rotary_frequencies(128, 1e6, {"type": "linear", "factor": 3.0})
    assert m == 1.0 and torch.allclose(g * 3, f, rtol=1e-14, atol=0)


def test_yarn_keeps_fast_pairs_and_interpolates_slow_ones():
    f, _ = rotary_frequencies(128, 1e6)
    g, m = rotary_frequencies(128, 1e6, YARN)
    turns = 32768 * f / (2 * math.pi)
    assert math.isclose(m, 0.1 * math.log(4.0) + 1)
    ratio = g / f
    # the borders are whole pairs outside the two turn counts
    assert (ratio[turns > 32 * (f[0] / f[1])] == 1).all()
    assert torch.allclose(ratio[turns < 1 / (f[0] / f[1])], torch.tensor(0.25, dtype=torch.float64))
    assert ((ratio[1:] - ratio[:-1]) <= 1e-15).all()
    assert rotary_frequencies(128, 1e6, dict(YARN, attention_factor=1.5))[1] == 1.5


def test_llama3_by_wave_length():
    f, _ = rotary_frequencies(64, 5e5)
    g, m = rotary_frequencies(64, 5e5, LLAMA3)
    wave = 2 * math.pi / f
    assert m == 1.0
    assert torch.equal(g[wave <= 8192 / 4], f[wave <= 8192 / 4])
    assert torch.allclose(g[wave >= 8192], f[wave >= 8192] / 8, rtol=1e-15)
    assert ((g <= f) & (g >= f / 8 * (1 - 1e-15))).all()


def test_dynamic_grows_the_base_beyond_the_trained_length():
    s = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 4096}
    f, _ = rotary_frequencies(64, 1e4)
    assert torch.equal(rotary_frequencies(64, 1e4, s)[0], f)
    assert torch.equal(rotary_frequencies(64, 1e4, s, seq_len=4096)[0], f)
    g, _ = rotary_frequencies(64, 1e4, s, seq_len=8192)
    base = 1e4 * 3.0 ** (64 / 62)
    assert math.isclose(float(g[-1]), base ** (-62 / 64), rel_tol=1e-12)
    # the slowest pair turns as far at 8192 as interpolation by 3 would have it
    assert math.isclose(float(g[-1] / f[-1]), 1 / 3.0, rel_tol=1e-12)


@pytest.mark.parametrize("scaling", [None, {"rope_type": "linear", "factor": 2.5}, YARN,
                                     dict(YARN, beta_fast=16, beta_slow=2), LLAMA3])
def test_against_transformers(scaling):
    """The library's own fp32 frequencies, run on the same configuration."""
    rope = pytest.importorskip("transformers.modeling_rope_utils")
    from transformers import Qwen3Config

    kind = (scaling or {"rope_type": "default"})["rope_type"]
    if kind not in rope.ROPE_INIT_FUNCTIONS:
        pytest.skip(f"{kind} not in this transformers")
    cfg = Qwen3Config(hidden_size=1024, num_attention_heads=16, head_dim=128, rope_theta=1e6,
                      max_position_embeddings=32768, rope_scaling=scaling)
    try:
        inv, m = rope.ROPE_INIT_FUNCTIONS[kind](cfg, device="cpu")
    except Exception as e:  # another version's calling convention
        pytest.skip(f"transformers' form is called another way: {e}")
    f, gain = rotary_frequencies(128, 1e6, scaling)
    # fp32 powers of 1e6 and a blend: a few units
    assert torch.allclose(inv.double(), f, rtol=2e-6, atol=0) and math.isclose(m, gain, rel_tol=1e-6)


def test_bad_scalings_are_refused():
    for bad in ({"rope_type": "linear"}, {"rope_type": "yarn", "factor": 4.0},
                {"rope_type": "no such thing", "factor": 2.0,
                 "original_max_position_embeddings": 10},
                {"rope_type": "linear", "factor": 0.5}, dict(LLAMA3, low_freq_factor=5.0)):
        with pytest.raises((ValueError, KeyError)):
            rotary_frequencies(128, 1e6, bad)
    for d in (0, -2, 7):
        with pytest.raises(ValueError):
            rotary_frequencies(d)
    with pytest.raises(ValueError):
        make_rotary(64, layout="neox")
    with pytest.raises(ValueError):
        Rotary(torch.ones(4))


def _s(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _rot(q=FAKE, qs=_s(2048, 128), k=FAKE, ks=_s(1024, 128), qo=FAKE, qos=_s(2048, 128), ko=FAKE,
         kos=_s(1024, 128), dt=0, inv=FAKE, f=1.0, lay=0, pos=FAKE, T=4, hq=16, hkv=8, D=128,
         r=128):
    return _lib.load().qwen3_rotary(q, qs, k, ks, qo, qos, ko, kos, dt, inv, f, lay, 0, pos, T, hq,
                                    hkv, D, r, None)


@pytest.mark.parametrize("code,over", [
    (-1, dict(q=None)), (-1, dict(qs=None)), (-1, dict(k=None)), (-1, dict(ko=None)),
    (-1, dict(ks=None)), (-1, dict(kos=None)), (-1, dict(qo=None)), (-1, dict(inv=None)),
    (-1, dict(pos=None)), (-3, dict(dt=3)), (-3, dict(dt=-1)), (-1, dict(lay=2)),
    (-3, dict(D=132)), (-3, dict(r=24)), (-3, dict(r=144)), (-3, dict(r=0)),
    (-3, dict(D=1024, r=528)), (-1, dict(hq=0)), (-1, dict(hkv=0)), (-1, dict(T=-1)),
    (-1, dict(hq=1 << 20)), (-1, dict(f=0.0)), (-1, dict(f=float("nan"))),
    (-1, dict(f=float("inf"))), (-2, dict(q=FAKE + 4)), (-2, dict(ko=FAKE + 2)),
    (-2, dict(qs=_s(2052, 128))), (-2, dict(kos=_s(1024, 4))), (0, dict(T=0)),
    (-2, dict(dt=2, qs=_s(2050, 128))),
])
def test_rotary_refuses(code, over):
    assert _rot(**over) == code, _lib.load().qwen3_attn_last_error()


def test_pool_forms_refuse():
    lib = _lib.load()
    s2, s4 = _s(2048, 128), _s(65536, 32768, 2048, 128)

    def slots(q=FAKE, k=FAKE, v=FAKE, slots=FAKE, kc=FAKE, layer=0, nb=8, bs=16, r=128, pos=FAKE):
        return lib.qwen3_rotary_slots_bf16(q, s2, k, s2, v, s2, FAKE, s2, None, None, FAKE, 1.0, 0,
                                           pos, slots, kc, s4, FAKE, s4, nb, layer, 2, 3, 16, 8,
                                           128, r, bs, None)

    for over in (dict(q=None), dict(k=None), dict(v=None), dict(slots=None), dict(kc=None),
                 dict(layer=2), dict(layer=-1), dict(nb=0), dict(bs=0), dict(pos=None)):
        assert slots(**over) == -1, over
    assert slots(r=20) == -3 and slots(v=FAKE + 8) == -2

    def decode(B=2, sl=FAKE, bt=FAKE, stride=8, rows=4, pages=8, layer=0, v=FAKE):
        return lib.qwen3_rotary_decode_bf16(FAKE, s2, FAKE, s2, v, s2, FAKE, s2, FAKE, 1.0, 0, FAKE,
                                            s4, FAKE, s4, 8, layer, 2, sl, bt, stride, rows, pages,
                                            None, None, B, 16, 8, 128, 128, 16, None)

    for over in (dict(B=-1), dict(sl=None), dict(bt=None), dict(stride=7), dict(rows=0),
                 dict(pages=0), dict(layer=2), dict(v=None)):
        assert decode(**over) == -1, over
    assert decode(B=0) == 0


def test_wrappers_refuse():
    rot = make_rotary(128)
    q, k = torch.zeros(3, 4, 128, dtype=torch.bfloat16), torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    pos = torch.arange(3)
    kb = torch.zeros(2, 1, 2, 16, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        rotary_embedding_hip(q, k, pos, rot)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        rotary_embedding_prefill_hip(q, k, k, pos, rot, pos, kb, kb, 0)
    for call in (lambda: rotary_embedding_hip(q.double(), None, pos, rot),
                 lambda: rotary_embedding_hip(q, k.float(), pos, rot),
                 lambda: rotary_embedding_hip(q, k, pos[:2], rot),
                 lambda: rotary_embedding_hip(q, k, pos.int(), rot),
                 lambda: rotary_embedding_hip(q[:, :, :64], None, pos, rot),
                 lambda: rotary_embedding_hip(q, k, pos, rot, q_out=k),
                 lambda: rotary_embedding_hip(q, None, pos, rot, k_out=k),
                 lambda: rotary_embedding_hip(q.transpose(1, 2), None, pos, rot),
                 lambda: rotary_embedding_prefill_hip(q.float(), k.float(), k.float(), pos, rot, pos,
                                                      kb, kb, 0),
                 lambda: rotary_embedding_prefill_hip(q, k, k, pos, rot, pos, kb[:, :, :1],
                                                      kb[:, :, :1], 0)):
        with pytest.raises(AssertionError):
            call()


def test_tables_and_config_take_scalings(tmp_path):
    import json

    from qwen3_engine_from_scratch_amd.config import Qwen3Config
    from qwen3_engine_from_scratch_amd.kernels.pre_attention import rope_tables

    plain = rope_tables(64, 1e4, 300)
    for none in (None, {"rope_type": "default"}):
        for a, b in zip(rope_tables(64, 1e4, 300, scaling=none), plain):
            assert torch.equal(a, b)
    cos, sin = rope_tables(128, 1e6, 5000, scaling=YARN)
    f, m = rotary_frequencies(128, 1e6, YARN)
    t = 4999 * f
    assert cos.shape == sin.shape == (5000, 128) and cos.dtype == torch.float32
    for table, fn in ((cos, torch.cos), (sin, torch.sin)):
        assert torch.equal(table[4999], (fn(t) * m).float().repeat(2))
    d = dict(hidden_size=64, num_attention_heads=2, num_key_value_heads=1, head_dim=32,
             num_hidden_layers=1, vocab_size=10, intermediate_size=64, rms_norm_eps=1e-6,
             rope_theta=1e4, rope_scaling=YARN)
    (tmp_path / "config.json").write_text(json.dumps(d))
    assert Qwen3Config.from_pretrained(str(tmp_path)).rope_scaling is None
    assert Qwen3Config.from_pretrained(str(tmp_path), use_rope_scaling=True).rope_scaling == YARN


def test_a_grid_beyond_32_bits_is_refused():
    assert _rot(T=1 << 33) == -1
    assert b"too many tokens" in _lib.load().qwen3_attn_last_error()
