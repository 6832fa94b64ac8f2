"""Rotary positions on the gfx950 HIP kernels: half or interleaved pairs, a whole
head or its first part, frequencies scaled for long contexts, with or without the
write of k and v into the paged pool (include/qwen3_attn.h).

The reference rotates from fp32 tables of the positions it allows
(qwen3/rope.py:42-110); the fused QK-norm step (kernels/pre_attention.py) keeps
those.  Here the angle is formed in 64 bits from the position itself, so a position
needs no table and a far one loses nothing.
"""
from __future__ import annotations

import functools
import math
from dataclasses import dataclass

import torch

from .. import _lib

__all__ = ["Rotary", "rotary_frequencies", "make_rotary", "rotary_embedding_hip",
           "rotary_embedding_prefill_hip", "rotary_embedding_decode_hip"]

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_LAYOUTS = {"half": 0, "interleaved": 1}


def rotary_frequencies(rotary_dim: int, base: float = 1e6, scaling: dict | None = None,
                       seq_len: int | None = None) -> tuple[torch.Tensor, float]:
    """Angular frequencies (rotary_dim / 2,) in float64 on the CPU and the factor on
    cos and sin.  scaling: None, or a rope_scaling dict of a model's config.json, by
    its "rope_type" (or "type"):

      default  f_i = base^(-2 i / rotary_dim)
      linear   f_i / factor
      dynamic  the base grows with seq_len beyond original_max_position_embeddings L:
               base * (factor seq_len / L - factor + 1)^(d / (d - 2))
      yarn     pairs that turn more than beta_fast times within L keep f_i, those that
               turn less than beta_slow times take f_i / factor, linear in i between;
               cos and sin times attention_factor (default m(1), or m(mscale) /
               m(mscale_all_dim) where both are given, m(k) = 0.1 k ln(factor) + 1)
      llama3   by wave length: f_i from L / high_freq_factor down, f_i / factor from
               L / low_freq_factor up, linear in L / wave length between

    A key that its type does not know is refused: it would ask for other angles.
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim {rotary_dim} must be positive and even")
    d = rotary_dim
    i = torch.arange(d // 2, dtype=torch.float64)
    freq = torch.pow(torch.tensor(float(base), dtype=torch.float64), -2 * i / d)
    scaling = dict(scaling or {})
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    _check_keys(scaling, kind, base)
    if kind == "default":
        return freq, 1.0
    factor = float(scaling["factor"])
    if not factor >= 1.0 or math.isinf(factor):
        raise ValueError(f"rope_scaling factor {factor} must be finite and at least 1")
    if kind == "linear":
        return freq / factor, 1.0
    L = scaling.get("original_max_position_embeddings")
    if L is None or not float(L) > 0:
        raise ValueError(f"rope_scaling {kind!r} needs original_max_position_embeddings")
    L = float(L)
    if kind == "dynamic":
        if seq_len is not None and seq_len > L:
            if d == 2:
                raise ValueError("dynamic scaling needs rotary_dim above 2")
            grown = base * (factor * seq_len / L - (factor - 1)) ** (d / (d - 2))
            return rotary_frequencies(d, grown)
        return freq, 1.0
    if kind == "yarn":
        def pair_turning(n):  # the (real) index whose pair turns n times within L
            return d * math.log(L / (2 * math.pi * n)) / (2 * math.log(base))

        low = pair_turning(float(scaling.get("beta_fast") or 32.0))
        high = pair_turning(float(scaling.get("beta_slow") or 1.0))
        if scaling.get("truncate", True):
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, d - 1)
        slow = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return freq * (1 - slow) + freq / factor * slow, _yarn_factor(scaling, factor)
    # llama3
    lo, hi = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
    if not 0 < lo < hi:
        raise ValueError("llama3 scaling needs 0 < low_freq_factor < high_freq_factor")
    keep = ((L * freq / (2 * math.pi) - lo) / (hi - lo)).clamp(0, 1)
    return freq * keep + freq / factor * (1 - keep), 1.0


# What a rope_scaling dict of each type may say, beside the keys of all of them.
_SCALING_KEYS = {
    "default": set(),
    "linear": {"factor"},
    "dynamic": {"factor"},
    "yarn": {"factor", "beta_fast", "beta_slow", "truncate", "attention_factor", "mscale",
             "mscale_all_dim"},
    "llama3": {"factor", "low_freq_factor", "high_freq_factor"},
}


def _check_keys(scaling: dict, kind, base: float) -> None:
    if kind not in _SCALING_KEYS:
        raise ValueError(f"rope_scaling type {kind!r} not supported")
    # these may come along, where they agree with what the caller says
    same = {"rope_type": kind, "type": kind, "rope_theta": base, "partial_rotary_factor": 1.0}
    for key, value in scaling.items():
        if value is None or key in _SCALING_KEYS[kind] or key == "original_max_position_embeddings":
            continue
        if key not in same:
            raise ValueError(f"rope_scaling key {key!r} is not one of type {kind!r}")
        if value != same[key]:
            raise ValueError(f"rope_scaling {key} {value!r} where {same[key]!r} is asked for")


def _yarn_factor(scaling: dict, factor: float) -> float:
    """yarn's factor on cos and sin."""
    if scaling.get("attention_factor") is not None:
        return float(scaling["attention_factor"])

    def m(k):
        return 0.1 * k * math.log(factor) + 1.0

    scales = [scaling.get("mscale"), scaling.get("mscale_all_dim")]
    if scales == [None, None]:
        return m(1.0)
    # one without the other, or a zero, means different things to different libraries
    if None in scales or not all(float(x) > 0 for x in scales):
        raise ValueError("yarn scaling takes mscale and mscale_all_dim together, both positive")
    return m(float(scales[0])) / m(float(scales[1]))


@dataclass(frozen=True)
class Rotary:
    """What a model keeps for its rotary positions: the frequencies on the device
    (float64, rotary_dim / 2), how elements pair up ("half": i with i + rotary_dim / 2,
    "interleaved": 2 i with 2 i + 1) and the factor on cos and sin."""
    inv_freq: torch.Tensor
    layout: str = "half"
    attention_factor: float = 1.0

    def __post_init__(self):
        if self.layout not in _LAYOUTS:
            raise ValueError(f"layout {self.layout!r}: half or interleaved")
        if self.inv_freq.dtype != torch.float64 or self.inv_freq.dim() != 1 \
                or not self.inv_freq.is_contiguous():
            raise ValueError("inv_freq must be a contiguous float64 vector")

    @functools.cached_property
    def rotary_dim(self) -> int:
        return 2 * self.inv_freq.numel()


def make_rotary(rotary_dim: int, base: float = 1e6, *, layout: str = "half",
                scaling: dict | None = None, seq_len: int | None = None, device=None) -> Rotary:
    """rotary_frequencies on a device."""
    freq, gain = rotary_frequencies(rotary_dim, base, scaling, seq_len)
    return Rotary(freq.to(device), layout, gain)


@functools.lru_cache(maxsize=1024)
def _layout(q, q_stride, q_type, k, k_stride, k_type, rotary_dim):
    """The checks that go by shapes, strides and types alone (kept by those); returns
    (tokens, query heads, KV heads, head_dim)."""
    assert len(q) == 3 and q_stride[2] == 1, "q must be (tokens, heads, head_dim) rows"
    assert q_type in _DTYPES, f"dtype {q_type} not supported"
    T, Hq, D = q
    if k is not None:
        assert len(k) == 3 and k_stride[2] == 1 and k_type == q_type
        assert k[0] == T and k[2] == D
    assert rotary_dim <= D, f"rotary_dim {rotary_dim} of head_dim {D}"
    return T, Hq, 0 if k is None else k[1], D


def _check(q, k, rotary, q_out, k_out):
    if k is None:
        assert k_out is None
        sizes = _layout(q.shape, q.stride(), q.dtype, None, None, None, rotary.rotary_dim)
    else:
        sizes = _layout(q.shape, q.stride(), q.dtype, k.shape, k.stride(), k.dtype,
                        rotary.rotary_dim)
        assert k_out is None or _like(k, k_out), "an output must have its input's shape and type"
    assert q_out is None or _like(q, q_out), "an output must have its input's shape and type"
    return sizes


def _like(x, y):
    return y.shape == x.shape and y.dtype == x.dtype and y.stride(2) == 1


def _positions(positions, T):
    assert positions.dtype == torch.int64 and positions.numel() == T
    return positions.contiguous()


def rotary_embedding_hip(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
                         rotary: Rotary, *, inverse: bool = False,
                         q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """q (T, Hq, D) and k (T, Hkv, D) (or None) rotated at positions (T,) int64, each of
    magnitude below 2^31; bf16, fp16 or fp32, views with strides welcome (slices of a
    fused projection).  Returns (q_out, k_out); they may be given, also as q and k
    themselves.  inverse: the transposed map, which takes the gradient of the outputs to
    that of the inputs; inputs that require a gradient get it (into outputs of the call's
    own)."""
    if _wants_grad(q, k):
        if q_out is not None or k_out is not None:
            raise RuntimeError("outputs that are given would lose the gradient of q and k: "
                               "leave them out, or call under torch.no_grad()")
        return _Rotated.apply(q, k, positions, rotary, inverse)
    return _rotate(q, k, positions, rotary, inverse, q_out, k_out)


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class _Rotated(torch.autograd.Function):
    """The map is linear and its transpose the inverse form: that is its gradient."""

    @staticmethod
    def forward(ctx, q, k, positions, rotary, inverse):
        ctx.rotary, ctx.inverse = rotary, inverse
        ctx.save_for_backward(positions)
        return _rotate(q, k, positions, rotary, inverse, None, None)

    @staticmethod
    def backward(ctx, gq, gk):
        positions, = ctx.saved_tensors
        grads = [_rows(g) if need else None for g, need in zip((gq, gk), ctx.needs_input_grad)]
        if grads[0] is None:  # k's alone
            dk, dq = rotary_embedding_hip(grads[1], None, positions, ctx.rotary,
                                          inverse=not ctx.inverse)
        else:
            dq, dk = rotary_embedding_hip(*grads, positions, ctx.rotary, inverse=not ctx.inverse)
        return dq, dk, None, None, None


def _rows(g: torch.Tensor) -> torch.Tensor:
    """A gradient as the kernel reads it: rows of 16-byte chunks, whatever it was."""
    chunk = 16 // g.element_size()
    ok = g.stride(2) == 1 and g.data_ptr() % 16 == 0 and all(s % chunk == 0 for s in g.stride()[:2])
    return g if ok else g.clone(memory_format=torch.contiguous_format)


def _rotate(q, k, positions, rotary, inverse, q_out, k_out):
    T, Hq, Hkv, D = _check(q, k, rotary, q_out, k_out)
    positions = _positions(positions, T)
    dev = _lib.require_hip(q, k, positions, rotary.inv_freq, q_out, k_out)
    q_out = torch.empty_like(q) if q_out is None else q_out
    if k is not None and k_out is None:
        k_out = torch.empty_like(k)
    if T == 0:
        return q_out, k_out
    st = _lib.outer_strides
    with _lib.on_device(dev):
        rc = _lib.load().qwen3_rotary(
            q.data_ptr(), st(q), _lib.ptr(k), None if k is None else st(k),
            q_out.data_ptr(), st(q_out), _lib.ptr(k_out),
            None if k is None else st(k_out), _DTYPES[q.dtype],
            rotary.inv_freq.data_ptr(), float(rotary.attention_factor), _LAYOUTS[rotary.layout],
            1 if inverse else 0, positions.data_ptr(), T, Hq, Hkv, D,
            rotary.rotary_dim, _lib.stream_of(dev))
    _lib.check(rc, "qwen3_rotary")
    return q_out, k_out


def _check_pool(q, k, v, k_buffer, v_buffer):
    if _wants_grad(q, k, v):
        raise RuntimeError("what is written into the pool has no gradient: call under "
                           "torch.no_grad(), or rotate with rotary_embedding_hip")
    assert v.dim() == 3 and v.stride(2) == 1 and v.shape == k.shape
    assert q.dtype == v.dtype == k_buffer.dtype == v_buffer.dtype == torch.bfloat16, "bf16 only"
    assert k_buffer.dim() == 5 and v_buffer.shape == k_buffer.shape
    assert k_buffer.shape[2] == k.shape[1] and k_buffer.shape[4] == k.shape[2]
    assert k_buffer.stride(4) == 1 and v_buffer.stride(4) == 1


def rotary_embedding_prefill_hip(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                                 positions: torch.Tensor, rotary: Rotary,
                                 slot_mapping: torch.Tensor, k_buffer: torch.Tensor,
                                 v_buffer: torch.Tensor, layer_idx: int, *,
                                 q_out: torch.Tensor | None = None,
                                 k_out: torch.Tensor | None = None):
    """rotary_embedding_hip of T packed tokens that also writes the rotated k and v
    into layer layer_idx of the pool at slot_mapping (T,) (int64 block * block_size +
    offset; negative: not written).  bf16.  Returns (q_out, k_out)."""
    T, Hq, Hkv, D = _check(q, k, rotary, q_out, k_out)
    _check_pool(q, k, v, k_buffer, v_buffer)
    positions = _positions(positions, T)
    slot_mapping = _positions(slot_mapping, T)
    dev = _lib.require_hip(q, k, v, positions, slot_mapping, rotary.inv_freq, k_buffer, v_buffer,
                           q_out, k_out)
    q_out = torch.empty_like(q) if q_out is None else q_out
    k_out = torch.empty_like(k) if k_out is None else k_out
    if T == 0:
        return q_out, k_out
    st = _lib.outer_strides
    with _lib.on_device(dev):
        rc = _lib.load().qwen3_rotary_slots_bf16(
            q.data_ptr(), st(q), k.data_ptr(), st(k), v.data_ptr(),
            st(v), q_out.data_ptr(), st(q_out), k_out.data_ptr(),
            st(k_out), rotary.inv_freq.data_ptr(), float(rotary.attention_factor),
            _LAYOUTS[rotary.layout], positions.data_ptr(), slot_mapping.data_ptr(),
            k_buffer.data_ptr(), st(k_buffer), v_buffer.data_ptr(),
            st(v_buffer), k_buffer.shape[0], int(layer_idx), k_buffer.shape[1], T,
            Hq, Hkv, D, rotary.rotary_dim, k_buffer.shape[3], _lib.stream_of(dev))
    _lib.check(rc, "qwen3_rotary_slots_bf16")
    return q_out, k_out


def rotary_embedding_decode_hip(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rotary: Rotary,
                                pool, layer_idx: int, row_ids: torch.Tensor | None = None, *,
                                positions: torch.Tensor | None = None,
                                q_out: torch.Tensor | None = None) -> torch.Tensor:
    """One token a sequence: returns the rotated q (B, Hq, D) and writes the rotated k
    and v into `pool` (a KVCachePool) at position seq_lens[row], whose page must be
    reserved; rotated there too, or at positions (B,) int64.  row_ids: int32 (B,) rows of
    the block table (None: row b for token b).  bf16."""
    B, Hq, Hkv, D = _check(q, k, rotary, q_out, None)
    kb, vb = pool.k_buffer, pool.v_buffer
    _check_pool(q, k, v, kb, vb)
    if row_ids is not None:
        assert row_ids.dtype == torch.int32 and row_ids.numel() == B
        row_ids = row_ids.contiguous()
    if positions is not None:
        positions = _positions(positions, B)
    bt = pool.block_table_2d
    dev = _lib.require_hip(q, k, v, rotary.inv_freq, kb, bt, row_ids, positions, q_out)
    q_out = torch.empty_like(q) if q_out is None else q_out
    if B == 0:
        return q_out
    st = _lib.outer_strides
    with _lib.on_device(dev):
        rc = _lib.load().qwen3_rotary_decode_bf16(
            q.data_ptr(), st(q), k.data_ptr(), st(k), v.data_ptr(),
            st(v), q_out.data_ptr(), st(q_out), rotary.inv_freq.data_ptr(),
            float(rotary.attention_factor), _LAYOUTS[rotary.layout], kb.data_ptr(),
            st(kb), vb.data_ptr(), st(vb), kb.shape[0],
            int(layer_idx), kb.shape[1], pool.seq_lens.data_ptr(), bt.data_ptr(), bt.stride(0),
            bt.shape[0], bt.shape[1], _lib.ptr(row_ids), _lib.ptr(positions), B, Hq, Hkv,
            D, rotary.rotary_dim, kb.shape[3], _lib.stream_of(dev))
    _lib.check(rc, "qwen3_rotary_decode_bf16")
    return q_out
