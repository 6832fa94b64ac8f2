"""Rotary positions on the GPU against the definition in 64 bits: layouts, parts of a
head, types, far and negative positions, strides, in place, the inverse as transpose
and gradient, and the writes into the pool.

Bound, derived: the angle in turns is exact to 3 2^-53 of its size, then rounded to
fp32 (2^-25 of a turn, 1.9e-7 rad); cos and sin are off by two units at most
(1.2e-7), their products and the sum by three roundings (1.8e-7): together below
6e-7 (|x_a| + |x_b|) factor plus 3.4e-16 |pos f| of the same; and the output's half
step, eps / 2 of it, or half of the smallest subnormal where that is more: below the
smallest normal (2^-14 in fp16) the steps no longer shrink with the value."""
import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu


def reference(x, pos, rot, sign=1.0):
    """(y, slack): the definition in 64 bits, and the bound's part in |x|."""
    r, f = rot.rotary_dim, rot.inv_freq.double()
    t = pos.double()[:, None] * f[None]
    c, s = (torch.cos(t) * rot.attention_factor)[:, None], (sign * torch.sin(t)
                                                           * rot.attention_factor)[:, None]
    xd = x.double()
    y, slack = xd.clone(), torch.zeros_like(xd)
    ia = torch.arange(r // 2, device=x.device)
    a, b = (ia, ia + r // 2) if rot.layout == "half" else (2 * ia, 2 * ia + 1)
    y[..., a] = xd[..., a] * c - xd[..., b] * s
    y[..., b] = xd[..., b] * c + xd[..., a] * s
    size = (xd[..., a].abs() + xd[..., b].abs()) * rot.attention_factor \
        * (6e-7 + 3.4e-16 * t.abs())[:, None]
    slack[..., a], slack[..., b] = size, size
    return y, slack


def check(out, x, pos, rot, what, sign=1.0):
    y, slack = reference(x, pos, rot, sign)
    info = torch.finfo(out.dtype)
    half = (info.eps / 2 * (y.abs() + slack)).clamp(min=info.smallest_normal * info.eps / 2)
    over = (out.double() - y).abs() - (half + slack)
    print(f"[err] {what}: worst excess {over.max().item():.3e}", flush=True)
    assert over.max() <= 0, what
    assert torch.equal(out[..., rot.rotary_dim:], x[..., rot.rotary_dim:])


def make(T, heads, D, dtype, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn(T, heads, D, generator=g, device=dev).to(dtype)


def _positions(lo, hi, n, dev):
    return torch.randint(lo, hi, (n,), generator=torch.Generator().manual_seed(n)).to(dev)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,hq,hkv,D,r", [(1, 16, 8, 128, 128), (5, 3, 1, 80, 32), (67, 8, 8, 64, 16),
                                          (130, 4, 2, 256, 256), (9, 2, 2, 512, 512),
                                          (33, 5, 3, 72, 64), (1000, 2, 1, 128, 96)])
def test_against_its_definition(gpu, dtype, layout, T, hq, hkv, D, r):
    from qwen3_engine_from_scratch_amd.kernels.rotary import make_rotary, rotary_embedding_hip

    announce(f"rotary {dtype} {layout} T={T} heads {hq}/{hkv} {r} of {D}")
    rot = make_rotary(r, 1e4, layout=layout, device=gpu)
    q, k = make(T, hq, D, dtype, gpu, 1), make(T, hkv, D, dtype, gpu, 2)
    pos = _positions(-5000, 200000, T, gpu)
    keep = q.clone(), k.clone()
    qo, ko = rotary_embedding_hip(q, k, pos, rot)
    torch.cuda.synchronize()
    assert torch.equal(q, keep[0]) and torch.equal(k, keep[1])
    check(qo, q, pos, rot, "q")
    check(ko, k, pos, rot, "k")
    qi, none = rotary_embedding_hip(q, None, pos, rot, inverse=True)
    assert none is None
    check(qi, q, pos, rot, "q back", sign=-1.0)
    a, b = q.clone(), k.clone()
    rotary_embedding_hip(a, b, pos, rot, q_out=a, k_out=b)
    torch.cuda.synchronize()
    assert torch.equal(a, qo) and torch.equal(b, ko), "in place"


def test_far_positions_and_scaled_frequencies(gpu):
    from qwen3_engine_from_scratch_amd.kernels.rotary import make_rotary, rotary_embedding_hip

    far = torch.tensor([0, 1, 131071, 2 ** 24 + 1, 2 ** 31 - 1, -(2 ** 31) + 1], device=gpu)
    for scaling in (None, {"rope_type": "linear", "factor": 4.0},
                    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768},
                    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0,
                     "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}):
        announce(f"far positions, {scaling}")
        rot = make_rotary(128, scaling=scaling, device=gpu)
        for dtype in (torch.float32, torch.bfloat16):
            q, k = make(6, 4, 128, dtype, gpu, 3), make(6, 2, 128, dtype, gpu, 4)
            qo, ko = rotary_embedding_hip(q, k, far, rot)
            check(qo, q, far, rot, f"q {scaling}")
            check(ko, k, far, rot, f"k {scaling}")
            # at position 0: the factor alone
            assert torch.equal(qo[0], (q[0].float() * rot.attention_factor).to(dtype))


def test_position_zero_is_the_identity(gpu):
    from qwen3_engine_from_scratch_amd.kernels.rotary import make_rotary, rotary_embedding_hip

    announce("rotary: position 0; infinities and NaN stay in their pair")
    rot = make_rotary(64, device=gpu)
    q = make(3, 2, 128, torch.bfloat16, gpu)
    q[1, 0, 5], q[2, 1, 100] = float("nan"), float("inf")
    qo, _ = rotary_embedding_hip(q, None, torch.tensor([0, 7, 9], device=gpu), rot)
    assert torch.equal(qo[0], q[0])
    bad = ~torch.isfinite(qo)
    assert bad.nonzero().tolist() == [[1, 0, 5], [1, 0, 37], [2, 1, 100]]


def test_strided_slices(gpu):
    from qwen3_engine_from_scratch_amd.kernels.rotary import make_rotary, rotary_embedding_hip

    announce("rotary on slices of a fused projection, strided outputs")
    rot = make_rotary(64, layout="interleaved", device=gpu)
    qkv = make(21, 1, 10 * 128, torch.bfloat16, gpu, 5)[:, 0]
    q, k = qkv[:, :768].view(21, 6, 128), qkv[:, 768:1024].view(21, 2, 128)
    hold = torch.full((21, 3, 9, 128), 4.0, dtype=torch.bfloat16, device=gpu)
    pos = torch.arange(42, device=gpu)[::2] * 1000
    qo, ko = rotary_embedding_hip(q, k, pos, rot, q_out=hold[:, 1, :6], k_out=hold[:, 1, 7:])
    check(qo, q, pos, rot, "q")
    check(ko, k, pos, rot, "k")
    assert (hold[:, 0] == 4).all() and (hold[:, 2] == 4).all() and (hold[:, 1, 6] == 4).all()
    # head-major memory
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(rotary_embedding_hip(qt, None, pos, rot)[0], qo)
    e, _ = rotary_embedding_hip(q[:0], k[:0], pos[:0], rot)
    assert e.shape == (0, 6, 128)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_inverse_is_the_transpose_and_the_gradient(gpu, layout):
    from qwen3_engine_from_scratch_amd.kernels.rotary import make_rotary, rotary_embedding_hip

    announce(f"rotary {layout}: inverse against the transpose, and differences")
    rot = make_rotary(96, layout=layout, device=gpu, scaling={
        "rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 4096})
    x, g = make(40, 3, 128, torch.float32, gpu, 6), make(40, 3, 128, torch.float32, gpu, 7)
    pos = _positions(0, 30000, 40, gpu)
    y = rotary_embedding_hip(x, None, pos, rot)[0]
    gx = rotary_embedding_hip(g, None, pos, rot, inverse=True)[0]
    # <g, R x> = <R^T g, x>, each element within 6e-7 (|a| + |b|) factor + 2^-24: fifteen
    # thousand products, so far below 1e-3 of either side's sum of sizes
    lhs, rhs = (g.double() * y.double()).sum(), (gx.double() * x.double()).sum()
    size = (g.double().abs() * y.double().abs()).sum()
    assert (lhs - rhs).abs() <= 4e-6 * size
    # the map is linear: a difference of step 1 is the derivative, less the roundings of y
    for t, h, e in ((0, 0, 0), (7, 2, 50), (39, 1, 95), (20, 0, 127)):
        x2 = x.clone()
        x2[t, h, e] += 1
        y2 = rotary_embedding_hip(x2, None, pos, rot)[0]
        num = ((y2.double() - y.double()) * g.double()).sum()
        assert (num - gx[t, h, e].double()).abs() <= 1e-4


@pytest.mark.parametrize("layout,r", [("half", 128), ("interleaved", 64)])
def test_prefill_write(gpu, layout, r):
    from qwen3_engine_from_scratch_amd.kernels.rotary import (make_rotary, rotary_embedding_hip,
                                                              rotary_embedding_prefill_hip)

    announce(f"rotary {layout} {r} with slot writes")
    T, hq, hkv = 45, 6, 2
    rot = make_rotary(r, layout=layout, device=gpu)
    qkv = make(T, 1, (hq + 2 * hkv) * 128, torch.bfloat16, gpu, 8)[:, 0]
    q = qkv[:, :hq * 128].view(T, hq, 128)
    k = qkv[:, hq * 128:(hq + hkv) * 128].view(T, hkv, 128)
    v = qkv[:, (hq + hkv) * 128:].view(T, hkv, 128)
    pos = _positions(0, 40000, T, gpu)
    kb = torch.full((9, 3, hkv, 16, 128), 2.0, dtype=torch.bfloat16, device=gpu)
    vb = kb.clone()
    slots = torch.randperm(9 * 16, device=gpu)[:T]
    slots[3], slots[10], slots[11] = -1, 9 * 16, 2 ** 40
    qo, ko = rotary_embedding_prefill_hip(q, k, v, pos, rot, slots, kb, vb, 1)
    qr, kr = rotary_embedding_hip(q, k, pos, rot)
    assert torch.equal(qo, qr) and torch.equal(ko, kr)
    wk, wv = torch.full_like(kb, 2.0), torch.full_like(kb, 2.0)
    for t in range(T):
        s = int(slots[t])
        if 0 <= s < 9 * 16:
            wk[s // 16, 1, :, s % 16], wv[s // 16, 1, :, s % 16] = kr[t], v[t]
    assert torch.equal(kb, wk) and torch.equal(vb, wv)


def test_decode_write(gpu):
    from qwen3_engine_from_scratch_amd.PagedKVcache import KVCachePool, PagedKVCache
    from qwen3_engine_from_scratch_amd.kernels.rotary import (make_rotary,
                                                              rotary_embedding_decode_hip,
                                                              rotary_embedding_hip)

    announce("rotary decode form: write at the row's length")
    pool = KVCachePool(16, 2, 16, 2, 128, device=gpu, dtype=torch.bfloat16, max_seq_len=64,
                       max_requests=8)
    caches = [PagedKVCache(pool) for _ in range(4)]
    for c, n in zip(caches, (0, 15, 16, 40)):
        c.reserve_slots(n + 1)
        c.advance_seq_len(n)
    rows = torch.tensor([c.row_id for c in caches] + [99, 0], dtype=torch.int32, device=gpu)
    assert 0 not in [c.row_id for c in caches]  # row 0: no pages, length 0
    rot = make_rotary(128, device=gpu)
    q, k, v = (make(6, h, 128, torch.bfloat16, gpu, 9 + h) for h in (4, 2, 2))
    v = -k
    for given in (None, torch.tensor([5, 4, 3, 2, 1, 0], device=gpu)):
        pool.k_buffer.zero_()
        pool.v_buffer.zero_()
        out = rotary_embedding_decode_hip(q, k, v, rot, pool, 1, rows, positions=given)
        at = torch.tensor([0, 15, 16, 40, 0, 0], device=gpu) if given is None else given
        qr, kr = rotary_embedding_hip(q, k, at, rot)
        assert torch.equal(out, qr)
        wk, wv = torch.zeros_like(pool.k_buffer), torch.zeros_like(pool.v_buffer)
        for i, (c, n) in enumerate(zip(caches, (0, 15, 16, 40))):
            b = c.block_table[n // 16]
            wk[b, 1, :, n % 16], wv[b, 1, :, n % 16] = kr[i], v[i]
        assert torch.equal(pool.k_buffer, wk) and torch.equal(pool.v_buffer, wv)


def test_capture(gpu):
    from qwen3_engine_from_scratch_amd.kernels.rotary import make_rotary, rotary_embedding_hip

    announce("rotary captured and replayed at other positions")
    rot = make_rotary(128, device=gpu)
    q, k = make(7, 4, 128, torch.bfloat16, gpu, 1), make(7, 2, 128, torch.bfloat16, gpu, 2)
    pos = torch.zeros(7, dtype=torch.int64, device=gpu)
    rotary_embedding_hip(q, k, pos, rot)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qo, ko = rotary_embedding_hip(q, k, pos, rot)
    for i in range(3):
        pos.copy_(torch.arange(7, device=gpu) * 1000 * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        a, b = rotary_embedding_hip(q, k, pos, rot)
        assert torch.equal(qo, a) and torch.equal(ko, b)
        check(qo, q, pos, rot, f"replay {i}")
