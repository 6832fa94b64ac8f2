"""Batched token sampling on the GPU (reference: qwen3/sampling.py).

sample_tokens keeps the reference's signature and contract: logits (B, V),
temperature / top_k / top_p as scalars or per-row lists / tensors, returns
(B, 1) int64.  Rows with temperature <= 0 take the argmax; the rest draw from
softmax(logits / temperature) restricted to the top_k largest logits (all
when top_k <= 0) and, within them, to the leading tokens whose mass before
them is <= top_p.  The rows go through the sampling kernels
(qwen3_sample_ws_bf16: for batches of up to 128 rows two launches that
split each row over 2-8 workgroups, else one workgroup per row), or, when
all rows are greedy and the batch is larger, the argmax kernel; there is no
host round trip for per-row parameters given as device tensors.  The random
stream is the kernel's own (Philox4x32-10), so draws match the reference in
distribution, not token for token — as the reference's own Triton path does
against its torch path (qwen3/sampling.py:17-20).

token_logprobs (beyond the reference) says how probable given tokens are: their log
probabilities, the entropy of the distributions and the most likely tokens, with a
gradient for the logits.
"""
from __future__ import annotations

import functools
import math
from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .kernels.model_ops import argmax

__all__ = ["sample_tokens", "token_logprobs", "TokenLogprobs"]

_SEED_COUNTER = 0


def _next_seed() -> int:
    """A fresh seed per call when none is given (the reference's rule of a
    counter over torch.initial_seed(), qwen3/sampling.py:44-47)."""
    global _SEED_COUNTER
    _SEED_COUNTER += 1
    return (torch.initial_seed() + _SEED_COUNTER * 0x9E3779B1) & 0xFFFFFFFFFFFF


def _param(value, B: int, device, dtype) -> torch.Tensor:
    if isinstance(value, torch.Tensor):
        t = value.to(device=device, dtype=dtype)
        if t.ndim == 0:
            t = t.expand(B)
        return t.reshape(B).contiguous()
    if isinstance(value, (list, tuple)):
        return torch.tensor(value, device=device, dtype=dtype)
    return torch.full((B,), value, device=device, dtype=dtype)


def _all_greedy(temperature) -> bool:
    if isinstance(temperature, torch.Tensor):
        return temperature.device.type == "cpu" and bool((temperature <= 0).all())
    if isinstance(temperature, (list, tuple)):
        return all(float(t) <= 0 for t in temperature)
    return float(temperature) <= 0


_WORKSPACES: dict = {}
# Workspaces replaced by a larger one stay allocated until the process ends:
# a graph captured earlier holds the old address and may still be replayed.
_SUPERSEDED: list = []


def _workspace(dev, stream: int, B: int, V: int):
    """The parallel form's workspace for this device and stream (grown, never
    shrunk, never freed); None under graph capture when it would have to grow
    (the call then takes the single-workgroup form, which needs none)."""
    need = int(_lib.load().qwen3_sample_workspace_bytes(B, V))
    if need == 0:  # one part per row: the single-workgroup form
        return None
    key = (str(dev), stream)
    ws = _WORKSPACES.get(key)
    if ws is not None and ws.numel() >= need:
        return ws
    if torch.cuda.is_current_stream_capturing():
        return None
    if ws is not None:
        _SUPERSEDED.append(ws)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _WORKSPACES[key] = ws
    return ws


def sample_tokens(logits: torch.Tensor, temperature=0.0, top_k=0, top_p=1.0,
                  seed: int | None = None) -> torch.Tensor:
    """(B, V) bf16 logits -> (B, 1) int64 tokens (reference:
    qwen3/sampling.py:234-270)."""
    if logits.ndim != 2:
        raise ValueError(f"logits must be (B, V), got shape {tuple(logits.shape)}")
    assert logits.dtype == torch.bfloat16 and logits.stride(1) == 1
    B, V = logits.shape
    dev = _lib.require_hip(logits)
    stream = _lib.stream_of(dev)
    if _all_greedy(temperature):
        ws = _workspace(dev, stream, B, V)
        if ws is None:  # one workgroup per row: the argmax kernel
            return argmax(logits).view(B, 1)
        # a small batch: the parallel form's greedy path (no temperatures:
        # every row greedy), each row split over several workgroups
        out = torch.empty(B, dtype=torch.int64, device=dev)
        _lib.check(_lib.load().qwen3_sample_ws_bf16(
            logits.data_ptr(), logits.stride(0), B, V, None, None, None, 0, out.data_ptr(),
            ws.data_ptr(), ws.numel(), stream), "qwen3_sample_ws_bf16")
        return out.view(B, 1)
    t = _param(temperature, B, dev, torch.float32)
    k = _param(top_k, B, dev, torch.int32)
    p = _param(top_p, B, dev, torch.float32)
    if seed is None:
        seed = _next_seed()
    out = torch.empty(B, dtype=torch.int64, device=dev)
    ws = _workspace(dev, stream, B, V)
    rc = _lib.load().qwen3_sample_ws_bf16(
        logits.data_ptr(), logits.stride(0), B, V, t.data_ptr(), k.data_ptr(), p.data_ptr(),
        int(seed) & (2 ** 64 - 1), out.data_ptr(), None if ws is None else ws.data_ptr(),
        0 if ws is None else ws.numel(), stream)
    _lib.check(rc, "qwen3_sample_ws_bf16")
    return out.view(B, 1)


_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_GIVEN = 64  # given tokens a row
MAX_TOP = 64    # most likely tokens a row


class TokenLogprobs(NamedTuple):
    """What token_logprobs returns; what was not asked for is None."""
    logprobs: torch.Tensor | None      # fp32, of tokens' shape
    entropy: torch.Tensor | None       # fp32 (T,)
    top_ids: torch.Tensor | None       # int64 (T, n)
    top_logprobs: torch.Tensor | None  # fp32 (T, n)


@functools.lru_cache(maxsize=1024)
def _logprobs_workspace(*shape) -> int:
    return int(_lib.load().qwen3_token_logprobs_workspace_bytes(*shape))


def _given(tokens) -> int:
    """Given tokens a row."""
    return 0 if tokens is None else 1 if tokens.ndim == 1 else tokens.shape[1]


def _forward(logits, tokens, top_n, entropy, temperature, stats):
    """One call of the kernel: (logprobs, entropy, top_ids, top_logprobs, stats)."""
    T, V = logits.shape
    dev = logits.device
    lib = _lib.load()
    dtype = _DTYPES[logits.dtype]
    given = _given(tokens)
    f32 = dict(dtype=torch.float32, device=dev)
    lp = None if tokens is None else torch.empty(tokens.shape, **f32)
    ent = torch.empty(T, **f32) if entropy else None
    ids = torch.empty(T, top_n, dtype=torch.int64, device=dev) if top_n else None
    top = torch.empty(T, top_n, **f32) if top_n else None
    st = torch.empty(T, 2, **f32) if stats else None
    if T == 0:
        return lp, ent, ids, top, st
    need = _logprobs_workspace(T, V, dtype, top_n)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    ptr = _lib.ptr
    with _lib.on_device(dev):
        rc = lib.qwen3_token_logprobs(
            logits.data_ptr(), logits.stride(0), dtype, T, V, ptr(tokens), given, temperature,
            ptr(lp), ptr(ent), top_n, ptr(ids), ptr(top), ptr(st), ptr(ws), need,
            _lib.stream_of(dev))
    _lib.check(rc, "qwen3_token_logprobs")
    return lp, ent, ids, top, st


class _TokenLogprobs(torch.autograd.Function):
    """token_logprobs as a differentiable function of the logits."""

    @staticmethod
    def forward(ctx, logits, tokens, top_n, entropy, temperature):
        lp, ent, ids, top, stats = _forward(logits, tokens, top_n, entropy, temperature, True)
        ctx.save_for_backward(logits, tokens, ent, ids, stats)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        if ids is not None:
            ctx.mark_non_differentiable(ids)
        return lp, ent, ids, top

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_ent, _, g_top):
        logits, tokens, ent, ids, stats = ctx.saved_tensors
        if g_lp is None and g_ent is None and g_top is None:
            return None, None, None, None, None
        T, V = logits.shape
        dev = logits.device
        g_lp, g_ent, g_top = (None if g is None else g.to(torch.float32).contiguous()
                              for g in (g_lp, g_ent, g_top))
        grad = torch.empty(T, V, dtype=logits.dtype, device=dev)
        if T == 0:
            return grad, None, None, None, None
        ptr = _lib.ptr
        with _lib.on_device(dev):
            rc = _lib.load().qwen3_token_logprobs_grad(
                logits.data_ptr(), logits.stride(0), _DTYPES[logits.dtype], T, V, ptr(tokens),
                _given(tokens), ctx.temperature, ptr(ent),
                0 if ids is None else ids.shape[1], ptr(ids), stats.data_ptr(), ptr(g_lp),
                ptr(g_ent), ptr(g_top), grad.data_ptr(), V, _lib.stream_of(dev))
        _lib.check(rc, "qwen3_token_logprobs_grad")
        return grad, None, None, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None = None, *, top_n: int = 0,
                   entropy: bool = False, temperature: float = 1.0) -> TokenLogprobs:
    """How probable tokens are under softmax(logits / temperature), rows apart.

    logits:   (T, V) bf16, fp16 or fp32, unit last stride, rows any stride apart
    tokens:   (T,) or (T, K) int64, K up to 64: the tokens to look up.  A negative id
              is no token (its log probability is 0 and has no gradient), one of V or
              more gives NaN
    top_n:    the most likely tokens too, up to 64 (and V): by falling logit, the lower
              id first among equal ones
    entropy:  the distributions' entropy too (in nats)
    Returns TokenLogprobs; differentiable with respect to the logits (once), by the log
    probabilities, the entropy and the top log probabilities.  Logits of -inf have no
    mass; a row of nothing else, or with NaN or +inf, gives NaN.  Logits with a forward-mode
    tangent are refused (NotImplementedError).  (A backward pass is
    captured into a graph for logits made inside the capture, or a leaf of which no eager
    graph lives: torch ends the process otherwise, whatever the operator.)
    """
    if logits.ndim != 2:
        raise ValueError(f"logits must be (T, V), got shape {tuple(logits.shape)}")
    T, V = logits.shape
    if logits.dtype not in _DTYPES:
        raise ValueError(f"logits of {logits.dtype} not supported (bf16, fp16 or fp32)")
    if V == 0 or V > 1 << 30:
        raise ValueError(f"a vocabulary of {V} tokens")
    if V > 1 and logits.stride(1) != 1:
        raise ValueError("logits must have unit last stride")
    if T > 1 and logits.stride(0) < V:
        raise ValueError("logits' rows overlap")
    if tokens is not None:
        if tokens.dtype != torch.int64 or tokens.ndim not in (1, 2) or tokens.shape[0] != T:
            raise ValueError(f"tokens must be int64 (T,) or (T, K), got {tokens.dtype} "
                             f"{tuple(tokens.shape)} for {T} rows")
        if tokens.ndim == 2 and not 0 < tokens.shape[1] <= MAX_GIVEN:
            raise ValueError(f"{tokens.shape[1]} tokens a row (1 to {MAX_GIVEN})")
    top_n = int(top_n)
    if not 0 <= top_n <= min(MAX_TOP, V):
        raise ValueError(f"top_n {top_n} outside 0..{min(MAX_TOP, V)}")
    temperature = float(temperature)
    if not (temperature >= 1e-30 and math.isfinite(temperature)):
        raise ValueError(f"temperature {temperature} must be positive and finite")
    if tokens is None and not top_n and not entropy:
        raise ValueError("nothing asked for: no tokens, no top_n, no entropy")
    if forward_ad.unpack_dual(logits).tangent is not None:
        raise NotImplementedError("token_logprobs has no forward-mode derivative")
    _lib.require_hip(logits, tokens)
    if tokens is not None:
        tokens = tokens.contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobs.apply(logits, tokens, top_n, bool(entropy),
                                                   temperature))
    return TokenLogprobs(*_forward(logits, tokens, top_n, bool(entropy), temperature, False)[:4])
