"""Chunk attention of few packed rows holds its probabilities as the decode does, in 16
bits: over a handful of keys, where outputs are small against the values they are
weighted from, a single bf16 rounding of P would show."""
import pytest
import torch

from conftest import announce
from oracle.chunk import paged_chunk_ref
from test_chunk_gpu import make_case, run

pytestmark = pytest.mark.gpu

SCALE = 128 ** -0.5


def bound(t, ref, spread):
    """Of |out - o|, for n keys a row.  With A the largest sum_d |q_d k_d| scale:
      * a score is a sum of 128 products, off by 128 steps of 2^-23 of A at most (sums that
        cut off instead of rounding), scaled, less the maximum, each 2^-23 of 2 A, the
        exponential two units of 2^-23: a weight is off by delta = (128 + 8) 2^-23 A + 2^-22
        of itself, the quotient of two sums of weights by 2 delta spread;
      * P = hi + lo: lo is rounded to half a step of a value of at most half a step of P,
        2^-8 2^-8 = 2^-16 of P: 2^-16 spread;
      * fp32 sums of n terms, twice, and the quotient: (2 n + 4) 2^-23 spread;
      * the output rounded once: 2^-8 of a value with the errors above in it."""
    lens = t["cu"].diff() + t["seq_lens"][t["row_ids"].long()]
    n = int(lens.max())
    T = t["q"].shape[0]
    kc = t["k"].double().nan_to_num(0.0).abs().amax(dim=(0, 1, 2))  # (D,)
    A = float((t["q"].double().abs().view(T, -1, 128) * kc).sum(-1).max()) * SCALE
    delta = 136 * 2.0 ** -23 * A + 2.0 ** -22
    e = (2 * delta + 2.0 ** -16 + (2 * n + 4) * 2.0 ** -23) * spread
    return e + 2.0 ** -8 * (ref.abs() + e)


@pytest.mark.parametrize("chunks,ctxs,hq,hkv", [
    ([4] * 24, [1] * 24, 32, 8),
    ([5, 3, 1] * 9, [2, 0, 5] * 9, 16, 8),
    ([1] * 40, [1, 2, 3, 9] * 10, 32, 2),
])
def test_probabilities_keep_sixteen_bits(gpu, chunks, ctxs, hq, hkv):
    announce(f"chunk precision: {len(chunks)} sequences of {chunks[0]}, heads {hq}/{hkv}")
    t = make_case(chunks, ctxs, hq, hkv, 16, gpu, seed=len(chunks), std=0.25)
    out = run(t, gpu).double()
    ref, spread = paged_chunk_ref(t["q"], t["k"], t["v"], t["table"], t["seq_lens"], t["row_ids"],
                                  t["cu"], 16, SCALE)
    over = (out - ref).abs() - bound(t, ref, spread)
    print(f"[err] worst excess {over.max().item():.3e}", flush=True)
    assert over.max() <= 0


def test_single_tokens_agree_with_decode_to_a_step(gpu):
    """Decode and chunk of one token hold P in the same bits: both within the bound."""
    from qwen3_engine_from_scratch_amd.kernels.paged_attention import paged_attention_decode_hip

    announce("chunks of one token and paged decode, both with P in 16 bits")
    t = make_case([1] * 30, [1, 2, 6] * 10, 32, 8, 16, gpu, seed=3, std=0.25)
    args = (t["q"], t["k"], t["v"], t["table"].to(gpu), t["seq_lens"].to(gpu), t["row_ids"].to(gpu))
    out, dec = run(t, gpu).double(), paged_attention_decode_hip(*args, 16).double()
    ref, spread = paged_chunk_ref(t["q"], t["k"], t["v"], t["table"], t["seq_lens"], t["row_ids"],
                                  t["cu"], 16, SCALE)
    e = bound(t, ref, spread)
    assert ((dec - ref).abs() <= e).all() and ((out - ref).abs() <= e).all()
