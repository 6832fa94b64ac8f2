"""rope_scaling dicts of a model's configuration: the factors they ask for, those that are
refused, and what a table of fixed length can hold of them (CPU)."""
import math

import pytest
import torch

from qwen3_engine_from_scratch_amd.kernels.rotary import rotary_frequencies

YARN = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096,
        "beta_fast": 32, "beta_slow": 1}


@pytest.mark.parametrize("mscale,mscale_all_dim", [(0.707, 1.0), (1.0, 1.0), (1.0, 0.707), (2.0, 0.5)])
def test_yarn_factor_of_two_scales(mscale, mscale_all_dim):
    """m(factor, mscale) / m(factor, mscale_all_dim), m(s, k) = 0.1 k ln(s) + 1."""
    d = dict(YARN, mscale=mscale, mscale_all_dim=mscale_all_dim)
    f, gain = rotary_frequencies(64, 1e4, d)
    assert math.isclose(gain, (0.1 * mscale * math.log(40) + 1) / (0.1 * mscale_all_dim * math.log(40) + 1),
                        rel_tol=1e-14)
    assert torch.equal(f, rotary_frequencies(64, 1e4, YARN)[0])
    # a factor of its own goes before both
    assert rotary_frequencies(64, 1e4, dict(d, attention_factor=1.25))[1] == 1.25


@pytest.mark.parametrize("mscale,mscale_all_dim", [(0.707, 1.0), (1.0, 1.0), (1.0, 0.707), (None, None)])
def test_yarn_factor_against_transformers(mscale, mscale_all_dim):
    rope = pytest.importorskip("transformers.modeling_rope_utils")
    from transformers import Qwen3Config

    d = dict(YARN)
    if mscale is not None:
        d.update(mscale=mscale, mscale_all_dim=mscale_all_dim)
    cfg = Qwen3Config(hidden_size=1024, num_attention_heads=16, head_dim=64, rope_theta=1e4,
                      max_position_embeddings=163840, rope_scaling=dict(d))
    try:
        inv, m = rope.ROPE_INIT_FUNCTIONS["yarn"](cfg, device="cpu")
    except Exception as e:  # another version's calling convention
        pytest.skip(f"transformers' form is called another way: {e}")
    f, gain = rotary_frequencies(64, 1e4, d)
    # fp32 powers of 1e4 and a blend: a few units
    assert torch.allclose(inv.double(), f, rtol=2e-6, atol=0) and math.isclose(m, gain, rel_tol=1e-6)


@pytest.mark.parametrize("over", [dict(mscale=1.0), dict(mscale_all_dim=1.0),
                                  dict(mscale=1.0, mscale_all_dim=0.0),
                                  dict(mscale=0.0, mscale_all_dim=1.0),
                                  dict(mscale=-1.0, mscale_all_dim=1.0)])
def test_one_scale_alone_is_refused(over):
    with pytest.raises(ValueError, match="mscale"):
        rotary_frequencies(64, 1e4, dict(YARN, **over))


LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}


@pytest.mark.parametrize("bad", [
    {"rope_type": "default", "mrope_section": [16, 24, 24]},
    {"mrope_section": [16, 24, 24]},
    {"factor": 4.0},                                    # a factor of no type
    {"rope_type": "linear", "factor": 2.0, "beta_fast": 32},
    {"rope_type": "linear", "factor": 2.0, "attention_factor": 1.1},
    dict(YARN, long_factor=[1.0] * 32),
    dict(YARN, low_freq_factor=1.0),
    dict(LLAMA3, mscale=1.0, mscale_all_dim=1.0),
    dict(YARN, rope_theta=5e5),                         # another base than the one given
    dict(YARN, partial_rotary_factor=0.5),
    dict(YARN, type="linear"),                          # two types
])
def test_keys_that_are_not_understood_are_refused(bad):
    from qwen3_engine_from_scratch_amd.kernels.pre_attention import rope_tables

    with pytest.raises(ValueError, match="rope_scaling"):
        rotary_frequencies(128, 1e4, bad)
    with pytest.raises(ValueError, match="rope_scaling"):
        rope_tables(128, 1e4, 64, scaling=bad)


def test_keys_that_say_nothing_new_are_taken():
    for kind, d in (("linear", {"factor": 2.0, "original_max_position_embeddings": 4096}),
                    ("default", {}), ("dynamic", {"factor": 2.0,
                                                  "original_max_position_embeddings": 4096})):
        want = rotary_frequencies(64, 1e4, {"rope_type": kind, **d})
        for more in ({"type": kind}, {"rope_theta": 1e4}, {"partial_rotary_factor": 1.0},
                     {"beta_fast": None}):
            got = rotary_frequencies(64, 1e4, {"rope_type": kind, **d, **more})
            assert torch.equal(got[0], want[0]) and got[1] == want[1]
    assert torch.equal(rotary_frequencies(64, 1e4, {})[0], rotary_frequencies(64, 1e4)[0])


def test_a_table_of_fixed_length_holds_no_growing_base():
    """dynamic turns a sequence of up to L tokens by the plain frequencies and a longer one
    by others: a table beyond L would be wrong for one of them."""
    from qwen3_engine_from_scratch_amd.kernels.pre_attention import rope_tables
    from qwen3_engine_from_scratch_amd.model import RotaryEmbedding

    d = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 4096}
    plain = rope_tables(64, 1e4, 4096, scaling={"rope_type": "linear", "factor": 1.0})
    for n in (1000, 4096):
        for a, b in zip(rope_tables(64, 1e4, n, scaling=d), plain):
            assert torch.equal(a, b[:n])
    for n in (4097, 16384):
        with pytest.raises(ValueError, match="dynamic"):
            rope_tables(64, 1e4, n, scaling=d)
        with pytest.raises(ValueError, match="dynamic"):
            RotaryEmbedding(64, 1e4, n, scaling=d)
