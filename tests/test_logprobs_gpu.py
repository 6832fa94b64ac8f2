"""Log probabilities of given tokens, entropies, most likely tokens and the gradient
against their definitions in 64 bits (oracle/logprobs.py): types, odd vocabularies, parts,
masked rows, ties, NaN and infinities, strides, streams and graphs."""
import pytest
import torch

from conftest import announce
from oracle.logprobs import EPS, Rows, ranking

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def call(logits, tokens, **kw):
    from qwen3_engine_from_scratch_amd.sampling import token_logprobs

    return token_logprobs(logits, tokens, **kw)


def make(rows, vocab, dtype, seed=0, std=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g) * std).to(TYPES[dtype])


def check(logits, tokens, got, *, top_n=0, temperature=1.0, what=""):
    """Every output of rows that have a distribution; logits and tokens on the CPU."""
    r = Rows(logits, temperature)
    n = logits.shape[0]
    if tokens is not None:
        t = tokens.reshape(n, -1)
        want = r.logp.gather(1, t.clamp(0, logits.shape[1] - 1))
        off = (got.logprobs.cpu().double().reshape(n, -1) - want).abs()
        ok = torch.isfinite(want)
        bound = r.logprob_error(torch.where(ok, want, torch.zeros_like(want)))
        print(f"[err] {what}: logprobs {off[ok].max().item() if ok.any() else 0:.2e} "
              f"of {bound.max().item():.2e}", flush=True)
        assert (off[ok] <= bound[ok]).all(), what
        assert torch.equal(got.logprobs.cpu().reshape(n, -1)[~ok].double(), want[~ok]), what
    if got.entropy is not None:
        off = (got.entropy.cpu().double() - r.entropy).abs()
        print(f"[err] {what}: entropy {off.max().item():.2e} of "
              f"{r.entropy_error().max().item():.2e}", flush=True)
        assert (off <= r.entropy_error()).all(), what
    if top_n:
        ids = ranking(logits, top_n)
        assert torch.equal(got.top_ids.cpu(), ids), what
        want = r.logp.gather(1, ids)
        ok = torch.isfinite(want)
        off = (got.top_logprobs.cpu().double() - want).abs()
        assert (off[ok] <= r.logprob_error(torch.where(ok, want, torch.zeros_like(want)))[ok]).all(), what
        assert torch.equal(got.top_logprobs.cpu()[~ok].double(), want[~ok]), what


SHAPES = [
    # rows, vocabulary, type, given, top, temperature
    (1, 1, "bf16", 1, 1, 1.0), (3, 2, "fp32", 1, 2, 1.0), (5, 3, "fp16", 2, 3, 0.7),
    (4, 7, "bf16", 1, 7, 1.0), (4, 8, "fp16", 1, 5, 1.0), (4, 9, "bf16", 3, 9, 2.0),
    (2, 63, "fp32", 1, 63, 1.0), (7, 64, "bf16", 1, 64, 1.0), (9, 301, "fp16", 64, 20, 1.0),
    (3, 4095, "bf16", 1, 50, 1.0), (3, 4096, "bf16", 1, 50, 0.5), (3, 4097, "bf16", 1, 50, 1.0),
    (2, 2049, "fp32", 1, 64, 1.0), (1, 20011, "fp32", 4, 33, 1.3), (1, 151936, "bf16", 1, 5, 1.0),
    (17, 50021, "fp16", 1, 20, 1.0), (33, 151936, "bf16", 1, 20, 0.8), (70, 8191, "fp32", 2, 1, 1.0),
    (1100, 1500, "bf16", 1, 10, 1.0), (1030, 5003, "fp32", 1, 0, 1.0), (1, 400003, "bf16", 1, 64, 1.0),
]


@pytest.mark.parametrize("rows,vocab,dtype,given,top,temperature", SHAPES)
def test_against_the_definition(gpu, rows, vocab, dtype, given, top, temperature):
    what = f"{rows} x {vocab} {dtype}, {given} given, top {top}, T {temperature}"
    announce("logprobs " + what)
    x = make(rows, vocab, dtype, seed=vocab + rows)
    g = torch.Generator().manual_seed(rows)
    t = torch.randint(0, vocab, (rows, given), generator=g)
    t = t[:, 0] if given == 1 else t
    got = call(x.to(gpu), t.to(gpu), top_n=top, entropy=True, temperature=temperature)
    torch.cuda.synchronize()
    check(x, t, got, top_n=top, temperature=temperature, what=what)
    alone = call(x.to(gpu), t.to(gpu), temperature=temperature)
    assert torch.equal(alone.logprobs, got.logprobs) and alone.entropy is None and alone.top_ids is None


def special_rows(vocab, dtype, kind):
    x = make(6, vocab, dtype, seed=9)
    low = torch.finfo(x.dtype).min
    if kind == "few left (-inf)":
        keep = x[:, 5:vocab:vocab // 7].clone()
        x.fill_(float("-inf"))
        x[:, 5:vocab:vocab // 7] = keep
    elif kind == "few left (lowest)":
        keep = x[:, 5:vocab:vocab // 7].clone()
        x.fill_(low)
        x[:, 5:vocab:vocab // 7] = keep
    elif kind == "one left":
        x[:3].fill_(float("-inf"))
        x[:3, vocab // 2] = 3.0
    elif kind == "lowest everywhere":
        x.fill_(low)
        x[0, 3] = float("-inf")
    elif kind == "largest values":
        x.fill_(low)
        x[:, 2:vocab:5] = torch.finfo(x.dtype).max
    elif kind == "equal":
        x.fill_(1.5)
    elif kind == "zeros of both signs":
        x.fill_(-1.0)
        x[:, ::3] = 0.0
        x[:, ::2] = -0.0
    elif kind == "two values":
        x = torch.where(x > 4, 2.0, 1.0).to(x.dtype)
    elif kind == "rising":
        x = torch.arange(vocab).float().expand(6, -1).div(vocab / 64).to(x.dtype).contiguous()
    elif kind == "one thread's":  # the large ones all in pieces of one thread
        e = 4 if dtype == "fp32" else 8
        x -= 20
        mine = (torch.arange(vocab) // e) % 512 < 5
        x[:, mine] += 20 + torch.arange(int(mine.sum())).to(x.dtype) / 256
    return x


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("kind", ["few left (-inf)", "few left (lowest)", "one left",
                                  "lowest everywhere", "largest values", "equal",
                                  "zeros of both signs", "two values", "rising", "one thread's"])
def test_masked_rows_and_ties(gpu, dtype, kind):
    for vocab, copies in ((997, 1), (150001, 1), (30011, 200)):
        announce(f"logprobs {kind} {dtype} {vocab}")
        x = special_rows(vocab, dtype, kind)
        t = torch.tensor([5, 2, vocab - 1, 0, vocab // 2, 5 + vocab // 7])
        got = call(x.repeat(copies, 1).to(gpu), t.repeat(copies).to(gpu), top_n=20, entropy=True)
        torch.cuda.synchronize()
        one = type(got)(*(None if v is None else v[-6:] for v in got))
        check(x, t, one, top_n=20, what=f"{kind} {dtype} {vocab}")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("kind", ["few left (-inf)", "few left (lowest)", "one left", "equal",
                                  "two values", "rising", "one thread's"])
@pytest.mark.parametrize("copies,top", [(1, 9), (1, 64), (1, 3), (10, 64), (13, 20)])
def test_parts_lists_joined(gpu, dtype, kind, copies, top):
    """Rows of 2 to 16 parts, whose lists are joined by rank or head by head."""
    x = special_rows(30011, dtype, kind)
    t = torch.tensor([5, 2, 30010, 0, 15005, 4292])
    announce(f"logprobs {kind} {dtype}, {6 * copies} rows, top {top}")
    got = call(x.repeat(copies, 1).to(gpu), t.repeat(copies).to(gpu), top_n=top, entropy=True)
    torch.cuda.synchronize()
    for i in range(1, copies):
        assert torch.equal(got.top_ids[:6], got.top_ids[6 * i:6 * i + 6])
    check(x, t, type(got)(*(None if v is None else v[:6] for v in got)), top_n=top,
          what=f"{kind} {dtype} {copies} x {top}")


def test_rows_without_a_distribution(gpu):
    for vocab in (50, 40013):
        announce(f"logprobs without a distribution {vocab}")
        x = make(5, vocab, "fp32", seed=1)
        x[0].fill_(float("-inf"))
        x[1, 7] = float("nan")
        x[2, 9] = float("inf")
        x[3, 11] = float("inf")
        x[3, 30] = float("nan")
        x[3, 13] = -float("nan")
        t = torch.tensor([3, 3, 3, 3, 3])
        got = call(x.to(gpu), t.to(gpu), top_n=12, entropy=True)
        torch.cuda.synchronize()
        assert torch.isnan(got.logprobs[:4]).all() and torch.isnan(got.entropy[:4]).all()
        assert torch.equal(got.top_ids.cpu(), ranking(x, 12))
        assert torch.isnan(got.top_logprobs[:4]).all()
        check(x[4:], t[4:], type(got)(*(v[4:] for v in got)), top_n=12)


def test_ids_that_are_no_token(gpu):
    x = make(4, 1000, "bf16")
    t = torch.tensor([[1, -1], [-100, 2], [1000, 3], [1 << 40, -(1 << 40)]])
    got = call(x.to(gpu), t.to(gpu)).logprobs.cpu()
    want = Rows(x).logp
    assert got[0, 1] == 0 and got[1, 0] == 0 and got[3, 1] == 0
    assert torch.isnan(got[2, 0]) and torch.isnan(got[3, 0])
    for r, k, i in ((0, 0, 1), (1, 1, 2), (2, 1, 3)):
        assert abs(got[r, k].double() - want[r, i]) < 1e-5


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_strides_and_odd_starts(gpu, dtype):
    announce(f"logprobs strides {dtype}")
    base = make(9, 5020, dtype, seed=4).to(gpu)
    t = torch.randint(0, 5001, (9,), generator=torch.Generator().manual_seed(2))
    wide = torch.stack([t, t + 1], 1).to(gpu)
    for at in (0, 1, 2, 3, 7):
        x = base[:, at:at + 5001]
        got = call(x, wide[:, 0], top_n=9, entropy=True)
        check(x.cpu(), t, got, top_n=9, what=f"offset {at}")
    x = base[::2, 3:4]
    # (one token: 0 but for the rounding of its exponent, x c - R, which the bound counts)
    got = call(x, torch.zeros(5, dtype=torch.int64, device=gpu), top_n=1)
    check(x.cpu(), torch.zeros(5, dtype=torch.int64), got, top_n=1, what="one column")
    assert (got.logprobs <= 0).all()
    row = base[2:3, 5:]
    check(row.cpu(), t[:1], call(row, t[:1].to(gpu), top_n=3), top_n=3)


def test_no_rows(gpu):
    x = torch.empty(0, 50, dtype=torch.bfloat16, device=gpu)
    got = call(x, torch.empty(0, 2, dtype=torch.int64, device=gpu), top_n=4, entropy=True)
    assert got.logprobs.shape == (0, 2) and got.entropy.shape == (0,) and got.top_ids.shape == (0, 4)
    got = call(x, None, top_n=1)
    assert got.logprobs is None and got.entropy is None and got.top_logprobs.shape == (0, 1)


GRADS = [
    # rows, vocabulary, type, given, top, entropy, temperature
    (1, 1, "fp32", 1, 0, True, 1.0), (3, 3, "bf16", 2, 2, True, 0.8), (4, 9, "fp16", 1, 4, True, 1.0),
    (5, 129, "fp32", 3, 5, True, 1.3), (6, 16385, "bf16", 1, 0, False, 1.0),
    (3, 16384, "fp16", 1, 0, True, 1.0), (2, 40009, "fp32", 64, 64, True, 0.6),
    (40, 151936, "bf16", 1, 0, True, 1.0), (7, 33001, "bf16", 0, 3, False, 1.0),
    (7, 8195, "fp32", 0, 0, True, 2.0),
]


@pytest.mark.parametrize("rows,vocab,dtype,given,top,entropy,temperature", GRADS)
def test_gradient_against_the_formula(gpu, rows, vocab, dtype, given, top, entropy, temperature):
    what = f"{rows} x {vocab} {dtype}, {given} given, top {top}, entropy {entropy}, T {temperature}"
    announce("logprobs gradient " + what)
    x = make(rows, vocab, dtype, seed=vocab)
    gen = torch.Generator().manual_seed(5)
    t = torch.randint(0, vocab, (rows, given), generator=gen) if given else None
    if given > 1:
        t[:, 1] = t[:, 0]  # the same token twice
        t[0, 0] = -1
    leaf = x.to(gpu).requires_grad_(True)
    r = call(leaf, None if t is None else t.to(gpu), top_n=top, entropy=entropy, temperature=temperature)
    outs, grads = [], []
    def upstream(v):
        g = torch.randn(v.shape, generator=gen)
        outs.append(v)
        grads.append(g.to(gpu))
        return g
    g = upstream(r.logprobs) if given else None
    h = upstream(r.top_logprobs) if top else None
    ge = upstream(r.entropy) if entropy else None
    dx, = torch.autograd.grad(outs, [leaf], grads)
    torch.cuda.synchronize()
    assert dx.dtype == x.dtype and dx.shape == x.shape
    want, off = Rows(x, temperature).gradient(t, g, None if not top else r.top_ids.cpu(), h, ge)
    eps = torch.finfo(x.dtype)
    over = (dx.cpu().double() - want).abs() - (off + (want.abs() + off) * eps.eps / 2
                                              + eps.smallest_normal * eps.eps + 2.0 ** -126)
    print(f"[err] {what}: worst excess {over.max().item():.2e}", flush=True)
    assert (over <= 0).all(), what


def test_gradient_against_differences(gpu):
    """Central differences of the call itself along random directions v: with steps of h,
    the error is h^2 / 6 of the third derivative (at most 6 sum |v|^3 p-weighted, below 6
    max |v|^3) and the outputs' rounding over h."""
    announce("logprobs gradient against differences")
    rows, vocab, h = 4, 777, 2.0 ** -6
    x = make(rows, vocab, "fp32", seed=3, std=1.5)
    gen = torch.Generator().manual_seed(8)
    t = torch.randint(0, vocab, (rows, 2), generator=gen).to(gpu)
    w = torch.randn(rows, 2, generator=gen).to(gpu)

    def loss(z):
        r = call(z, t, entropy=True, top_n=3)
        return (r.logprobs.double() * w).sum() + 0.5 * r.entropy.double().sum() \
            + r.top_logprobs.double().sum()

    leaf = x.to(gpu).requires_grad_(True)
    loss(leaf).backward()
    for seed in range(4):
        v = (torch.rand(rows, vocab, generator=torch.Generator().manual_seed(seed)) - 0.5).to(gpu)
        with torch.no_grad():
            diff = (loss(leaf + h * v) - loss(leaf - h * v)) / (2 * h)
        along = (leaf.grad.double() * v).sum()
        weights = float(w.abs().sum()) + 0.5 * rows * 12 + 3 * rows
        # rounding: each output within 60 EPS of its value of about ten
        bound = weights * (h * h * 6 * 0.5 ** 3 + 60 * EPS * 10 / h)
        print(f"[err] difference {abs(float(diff - along)):.2e} of {bound:.2e}", flush=True)
        assert abs(float(diff - along)) < bound


def test_gradient_of_masked_rows(gpu):
    for kind in ("few left (-inf)", "one left", "lowest everywhere", "equal", "largest values"):
        announce(f"logprobs gradient {kind}")
        x = special_rows(2003, "fp32", kind)
        t = torch.full((6,), 5 if kind != "one left" else 1001)
        leaf = x.to(gpu).requires_grad_(True)
        r = call(leaf, t.to(gpu), entropy=True)
        g, ge = torch.linspace(-1, 1, 6), torch.full((6,), 0.3)
        dx, = torch.autograd.grad([r.logprobs, r.entropy], [leaf], [g.to(gpu), ge.to(gpu)])
        want, off = Rows(x).gradient(t, g, None, None, ge)
        over = (dx.cpu().double() - want).abs() - (off + want.abs() * 2.0 ** -24 + 2.0 ** -126)
        assert (over <= 0).all(), kind
    x = make(3, 100, "fp32")
    x[0].fill_(float("-inf"))
    x[1, 3] = float("nan")
    leaf = x.to(gpu).requires_grad_(True)
    call(leaf, torch.tensor([1, 1, 1], device=gpu)).logprobs.sum().backward()
    assert torch.isnan(leaf.grad[:2]).all() and torch.isfinite(leaf.grad[2]).all()


def test_gradient_uses(gpu):
    """Broadcast upstream gradients, one output used, strided logits, a gradient of no use."""
    base = make(6, 1030, "fp32").to(gpu).requires_grad_(True)
    t = torch.arange(6, device=gpu)
    r = call(base[:, 3:1010], t, entropy=True)
    r.logprobs.mean().backward()
    want, off = Rows(base.detach()[:, 3:1010].cpu()).gradient(t.cpu(), torch.full((6,), 1 / 6))
    assert ((base.grad[:, 3:1010].cpu().double() - want).abs() <= off + want.abs() * 2.0 ** -24 + 2.0 ** -126).all()
    assert not base.grad[:, :3].any() and not base.grad[:, 1010:].any()
    with torch.no_grad():
        assert not call(base, t).logprobs.requires_grad
    r = call(base, t, top_n=2)
    assert not r.top_ids.requires_grad and r.top_logprobs.requires_grad
    g, = torch.autograd.grad(r.logprobs.sum(), base, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_another_stream_and_a_graph(gpu):
    announce("logprobs on a stream and in a graph")
    x = make(3, 60013, "bf16", seed=2).to(gpu)
    t = torch.tensor([1, 2, 3], device=gpu)
    ref = call(x, t, top_n=7, entropy=True)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = call(x, t, top_n=7, entropy=True)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    static = x.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call(static, t, top_n=7, entropy=True)
    for seed in range(4):
        y = make(3, 60013, "bf16", seed=seed).to(gpu)
        static.copy_(y)
        g.replay()
        torch.cuda.synchronize()
        want = call(y, t, top_n=7, entropy=True)
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_gradient_in_a_graph(gpu):
    """Forward and backward captured, replayed with other logits and upstream gradients."""
    announce("logprobs: gradient captured")
    x = make(5, 4099, "bf16", seed=3).to(gpu)
    t = torch.tensor([[1, 2], [3, 3], [-1, 4098], [7, 0], [9, 4]], device=gpu)
    up = [torch.randn(5, 2, device=gpu), torch.randn(5, device=gpu), torch.randn(5, 3, device=gpu)]

    def step():
        leaf = x.detach().requires_grad_()
        r = call(leaf, t, top_n=3, entropy=True, temperature=0.7)
        return torch.autograd.grad([r.logprobs, r.entropy, r.top_logprobs], leaf, up)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        d = step()
    for i in range(4):
        x.copy_(make(5, 4099, "bf16", seed=20 + i))
        for u in up:
            u.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(d, step())


def test_logits_past_32_bits(gpu):
    """Rows whose bytes and elements lie past 2^32 and 2^31, of logits and gradient; strided."""
    announce("logprobs: 4.5 GB of logits")
    vocab, rows, stride = 151936, 15000, 152000
    x = torch.zeros(rows, stride, dtype=torch.bfloat16, device=gpu)[:, 8:8 + vocab]
    assert x.stride(0) * (rows - 1) > 2 ** 31
    last = make(5, vocab, "bf16", seed=5)
    x[-5:] = last.to(gpu)
    t = torch.zeros(rows, dtype=torch.long, device=gpu)
    t[-5:] = torch.tensor([0, 7, vocab - 1, 151000, 64], device=gpu)
    x.requires_grad_()
    r = call(x, t, top_n=3, entropy=True)
    end = type(r)(*(v.detach()[-5:] for v in r))
    check(last, t[-5:].cpu(), end, top_n=3, what="the last rows")
    up = torch.ones(rows, device=gpu)
    dx, = torch.autograd.grad(r.logprobs, x, up)
    alone = last.to(gpu).requires_grad_()
    few, = torch.autograd.grad(call(alone, t[-5:], top_n=3, entropy=True).logprobs, alone, up[-5:])
    assert (dx[-5:].float() - few.float()).abs().max() <= few.abs().max().float() * 2.0 ** -7
    assert not dx[:8, 1:].ne(dx[0, 1]).any()
