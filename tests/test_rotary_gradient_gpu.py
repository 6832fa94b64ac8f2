"""The gradient of rotary positions through autograd: the transposed map of the outputs'
gradient, against 64 bits and against differences of the outputs."""
import pytest
import torch

from conftest import announce
from test_rotary_gpu import _positions, check, make

pytestmark = pytest.mark.gpu


def _setup(gpu, dtype, layout="half", r=64, T=37, hq=4, hkv=2, D=128, scaling=None):
    from qwen3_engine_from_scratch_amd.kernels.rotary import make_rotary

    rot = make_rotary(r, 1e4, layout=layout, device=gpu, scaling=scaling)
    q, k = make(T, hq, D, dtype, gpu, 1), make(T, hkv, D, dtype, gpu, 2)
    gq, gk = make(T, hq, D, dtype, gpu, 3), make(T, hkv, D, dtype, gpu, 4)
    return rot, q, k, gq, gk, _positions(-500, 20000, T, gpu)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout,r", [("half", 128), ("interleaved", 32)])
@pytest.mark.parametrize("inverse", [False, True])
def test_gradient_is_the_transposed_map(gpu, dtype, layout, r, inverse):
    from qwen3_engine_from_scratch_amd.kernels.rotary import rotary_embedding_hip

    announce(f"rotary gradient {dtype} {layout} {r} inverse={inverse}")
    rot, q, k, gq, gk, pos = _setup(gpu, dtype, layout, r)
    want = rotary_embedding_hip(q, k, pos, rot, inverse=inverse)
    q.requires_grad_()
    k.requires_grad_()
    out = rotary_embedding_hip(q, k, pos, rot, inverse=inverse)
    assert all(torch.equal(a, b) and a.requires_grad for a, b in zip(out, want))
    dq, dk = torch.autograd.grad(out, (q, k), (gq, gk))
    torch.cuda.synchronize()
    sign = 1.0 if inverse else -1.0
    check(dq, gq, pos, rot, "dq", sign=sign)
    check(dk, gk, pos, rot, "dk", sign=sign)


def test_one_gradient_of_two_and_no_k(gpu):
    from qwen3_engine_from_scratch_amd.kernels.rotary import rotary_embedding_hip

    announce("rotary gradient: of q alone, of k alone, of one output, without k")
    rot, q, k, gq, gk, pos = _setup(gpu, torch.float32)
    for leaf, i, g in ((q, 0, gq), (k, 1, gk)):
        leaf.requires_grad_()
        out = rotary_embedding_hip(q, k, pos, rot)
        d, = torch.autograd.grad(out[i], leaf, g)
        check(d, g, pos, rot, f"output {i}", sign=-1.0)
        leaf.requires_grad_(False)
    q.requires_grad_()
    k.requires_grad_()
    dq, dk = torch.autograd.grad(rotary_embedding_hip(q, k, pos, rot)[0], (q, k), gq)
    check(dq, gq, pos, rot, "q of q", sign=-1.0)
    assert not dk.any()
    d, = torch.autograd.grad(rotary_embedding_hip(q, None, pos, rot)[0], q, gq)
    check(d, gq, pos, rot, "without k", sign=-1.0)


def test_strided_and_broadcast_gradients(gpu):
    """Gradients as autograd hands them on: a sum's (every stride zero), a slice of a wider
    one, one whose rows are not 16-byte aligned."""
    from qwen3_engine_from_scratch_amd.kernels.rotary import rotary_embedding_hip

    announce("rotary gradient: broadcast, strided and unaligned gradients")
    rot, q, k, gq, gk, pos = _setup(gpu, torch.bfloat16, r=128)
    qkv = torch.cat((q.flatten(1), k.flatten(1)), 1).requires_grad_()
    qs, ks = qkv[:, :512].view(37, 4, 128), qkv[:, 512:].view(37, 2, 128)
    (rotary_embedding_hip(qs, ks, pos, rot)[0].sum()
     + rotary_embedding_hip(qs, ks, pos, rot)[1].sum()).backward()
    ones = torch.ones_like(q)
    check(qkv.grad[:, :512].view(37, 4, 128), ones, pos, rot, "sum", sign=-1.0)
    check(qkv.grad[:, 512:].view(37, 2, 128), ones[:, :2], pos, rot, "sum", sign=-1.0)
    q.requires_grad_()
    wide = torch.zeros(37, 4, 133, dtype=torch.bfloat16, device=gpu)
    wide[:, :, 3:131] = gq
    for g in (wide[:, :, 3:131], gq.transpose(0, 1).contiguous().transpose(0, 1),
              gq.transpose(1, 2).contiguous().transpose(1, 2)):
        d, = torch.autograd.grad(rotary_embedding_hip(q, None, pos, rot)[0], q, g)
        check(d, gq, pos, rot, f"strides {g.stride()}", sign=-1.0)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_against_differences(gpu, layout):
    """The map is linear: <g, R(x + d)> - <g, R(x)> = <R^T g, d>, up to the roundings: each
    output off by 2^-24 of itself and 6e-7 (|x_a| + |x_b|) factor (test_rotary_gpu.py),
    the gradient the same in g; x + d is rounded once, 2^-24 of each element."""
    from qwen3_engine_from_scratch_amd.kernels.rotary import rotary_embedding_hip

    announce(f"rotary gradient against differences, {layout}")
    yarn = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}
    rot, q, _, g, _, pos = _setup(gpu, torch.float32, layout, 128, scaling=yarn)
    d = make(37, 4, 128, torch.float32, gpu, 9)
    q.requires_grad_()
    y, _ = rotary_embedding_hip(q, None, pos, rot)
    dq, = torch.autograd.grad(y, q, g)
    y2, _ = rotary_embedding_hip((q + d).detach(), None, pos, rot)
    lhs = (g.double() * (y2.double() - y.detach().double())).sum()
    rhs = (dq.double() * d.double()).sum()
    # one element's error at most: its own rounding and the bound's part, both sides of a
    # difference, with every |x| and |g| replaced by the largest and pairs by twice that
    big = max(float(t.abs().max()) for t in (q.detach(), q.detach() + d, d))
    step = (2.0 ** -24 * 2 + 6e-7 * 2 + 3.4e-16 * 20000 * 2) * rot.attention_factor * 2 * big
    assert abs(lhs - rhs) <= 3 * step * float(g.abs().sum()) + 2 * step * float(g.abs().max()) * d.numel()


def test_second_derivative_and_capture(gpu):
    from qwen3_engine_from_scratch_amd.kernels.rotary import rotary_embedding_hip

    announce("rotary gradient: through the gradient, and captured")
    rot, q, k, gq, gk, pos = _setup(gpu, torch.float32, r=128)
    q.requires_grad_()
    gq.requires_grad_()
    dq, = torch.autograd.grad(rotary_embedding_hip(q, None, pos, rot)[0], q, gq, create_graph=True)
    back, = torch.autograd.grad(dq, gq, q.detach())
    check(back, q.detach(), pos, rot, "second", sign=1.0)
    del dq, back
    q, gq = q.detach().clone(), gq.detach().clone()

    def step():
        x = q.detach().requires_grad_()
        return torch.autograd.grad(rotary_embedding_hip(x, None, pos, rot)[0], x, gq)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        d = step()
    for i in range(3):
        gq.copy_(make(37, 4, 128, torch.float32, gpu, 20 + i))
        graph.replay()
        torch.cuda.synchronize()
        check(d, gq, pos, rot, f"replay {i}", sign=-1.0)
        assert torch.equal(d, step())
