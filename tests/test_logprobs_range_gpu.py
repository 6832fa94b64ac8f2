"""Log probabilities, entropies, most likely tokens and gradients of rows whose scaled
logits lie far from zero -- finite masks, small temperatures, parts on both sides of the
border between the two forms of the sums -- against their definitions in 64 bits."""
import pytest
import torch

from conftest import announce
from oracle.logprobs import Rows, ranking
from test_logprobs_gpu import call, check, make

pytestmark = pytest.mark.gpu

BORDER = 2.0 ** 24 * 0.6931471805599453  # of |max| / temperature between the two forms


def far_rows(vocab, dtype, kind):
    """Six rows of a kind.  Whole columns are masked or lowered, so that parts (runs of
    columns) and threads (columns dealt in turn) meet them alone."""
    x = make(6, vocab, dtype, seed=vocab)
    col = torch.arange(vocab)
    if isinstance(kind, float):  # equal but for every 101st
        x.fill_(kind)
        x[:, 7::101] = kind - abs(kind) / 64
    elif kind.startswith("masked by"):
        keep = (col % 211 == 210) | (col >= vocab - 3)
        x[:, ~keep] = float(kind.split()[-1])
    elif kind == "falling":
        x = (x.float() - 10.0 ** (4 + 30 * col / vocab)).to(x.dtype)
    elif kind == "rising":
        x = (x.float() + 10.0 ** (4 + 30 * col / vocab)).to(x.dtype)
    elif kind in ("below the border", "above the border"):
        g = torch.Generator().manual_seed(3)
        steps = torch.randint(0, 4, (6, vocab), generator=g) + 4 * ((col // 1009) % 3)
        x = (steps.float() - 6 + round(BORDER) * (-1 if kind.startswith("below") else 1)).to(x.dtype)
    return x


FAR = [-1e10, -1e30, -3e38, 1e10, 1e30, 3e38, "masked by -1e9", "masked by -1e10", "masked by -1e30",
       "falling", "rising", "below the border", "above the border"]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("kind", FAR)
def test_far_logits(gpu, kind, dtype):
    if dtype == "bf16" and isinstance(kind, str) and kind.endswith("border"):
        dtype = "fp16"  # (bf16 has no steps of one there: ordinary rows, another type)
        kind = "masked by -6e4"
    for vocab, copies in ((8, 1), (997, 1), (150001, 1), (30011, 200)):
        what = f"{kind} {dtype} {vocab}"
        announce("logprobs far: " + what)
        x = far_rows(vocab, dtype, kind)
        t = torch.tensor([0, 2, vocab - 1, 7, vocab // 2, vocab // 3])
        top = min(20, vocab)
        got = call(x.repeat(copies, 1).to(gpu), t.repeat(copies).to(gpu), top_n=top, entropy=True)
        torch.cuda.synchronize()
        check(x, t, type(got)(*(v[-6:] for v in got)), top_n=top, what=what)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("temperature", [1e-4, 1e-6, 1e-7, 1e-9, 1e-10, 1e-20, 1e-30])
def test_small_temperatures(gpu, temperature, dtype):
    for vocab, copies in ((4, 1), (4099, 1), (60013, 1), (8009, 150)):
        what = f"T {temperature} {dtype} {vocab}"
        announce("logprobs far: " + what)
        x = make(6, vocab, dtype, seed=vocab)
        x[0] -= 30
        x[1, 1::2] = x[1, 0]
        x[2] = x[2, 0]
        if vocab == 4:
            x[3] = torch.tensor([20.125, 19.5, 3.0, 1.0])
        t = x.float().argmax(1)
        t[4] = vocab - 1
        top = min(9, vocab)
        got = call(x.repeat(copies, 1).to(gpu), t.repeat(copies).to(gpu), top_n=top, entropy=True,
                   temperature=temperature)
        torch.cuda.synchronize()
        check(x, t, type(got)(*(v[-6:] for v in got)), top_n=top, temperature=temperature, what=what)


@pytest.mark.parametrize("kind", FAR + ["T 1e-09", "T 1e-20"])
def test_gradient_of_far_logits(gpu, kind):
    for vocab in (8, 2003, 40009):
        what = f"{kind} {vocab}"
        announce("logprobs gradient far: " + what)
        temperature = 1.0
        if isinstance(kind, str) and kind.startswith("T "):
            temperature = float(kind.split()[1])
            x = make(6, vocab, "fp32", seed=vocab)
            x[1, 1::2] = x[1, 0]
            x[2] = x[2, 0]
        else:
            x = far_rows(vocab, "fp32", kind)
        t = torch.tensor([0, 2, vocab - 1, 7, vocab // 2, vocab // 3])
        leaf = x.to(gpu).requires_grad_(True)
        r = call(leaf, t.to(gpu), top_n=2, entropy=True, temperature=temperature)
        g, ge = torch.linspace(-1, 1, 6), torch.full((6,), 0.3)
        h = torch.tensor([[0.5, -0.25]]).repeat(6, 1)
        dx, = torch.autograd.grad([r.logprobs, r.entropy, r.top_logprobs], [leaf],
                                  [g.to(gpu), ge.to(gpu), h.to(gpu)])
        torch.cuda.synchronize()
        want, off = Rows(x, temperature).gradient(t, g, r.top_ids.cpu(), h, ge)
        # A probability below 2^-126 is zero in 32 bits, and the element's term of it,
        # p (sum g + sum h + g_H (log p + H)), with it: |log p| is below 104 down to the
        # least subnormal, from where on the exact term is smaller than 2^-149 times as much.
        size = g.abs() + h.abs().sum(1) + ge * (104 + Rows(x, temperature).entropy)
        gone = (2.0 ** -126 * size / temperature)[:, None]
        over = (dx.cpu().double() - want).abs() - (off + gone + want.abs() * 2.0 ** -24 + 2.0 ** -126)
        print(f"[err] {what}: worst excess {over.max().item():.2e}", flush=True)
        assert (over <= 0).all(), what


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_nan_at_the_first_tokens(gpu, dtype):
    """NaN at token 0, in every token, with as many listed as there are tokens."""
    for vocab, top in ((1, 1), (5, 5), (64, 64), (997, 12), (40013, 12), (150001, 64)):
        announce(f"logprobs NaN at token 0: {vocab} {dtype}, top {top}")
        x = make(4, vocab, dtype, seed=vocab)
        x[0, 0] = float("nan")
        x[1] = float("nan")
        x[2, ::3] = -float("nan")
        x[2, 1::3] = float("inf")
        x[3, -1] = float("nan")
        got = call(x.to(gpu), None, top_n=top)
        torch.cuda.synchronize()
        assert torch.equal(got.top_ids.cpu(), ranking(x, top))
        assert torch.isnan(got.top_logprobs).all()


@pytest.mark.parametrize("temperature", [1.0, 0.37, 1e-9])
def test_entropy_is_not_below_zero(gpu, temperature):
    """One token with all of the mass, in rows of one part and of several."""
    for rows, vocab in ((4096, 300), (40, 30011)):
        announce(f"logprobs: entropy of one token, {rows} x {vocab}, T {temperature}")
        x = torch.full((rows, vocab), float("-inf"))
        x[:, 5] = torch.linspace(-900, 900, rows)
        peaked = make(rows, vocab, "fp32", seed=3, std=60.0)
        for y in (x, peaked):
            got = call(y.to(gpu), None, entropy=True, temperature=temperature)
            torch.cuda.synchronize()
            assert (got.entropy >= 0).all()
            check(y[:50], None, type(got)(*(v if v is None else v[:50] for v in got)),
                  temperature=temperature, what=f"entropy {rows} x {vocab}")


@pytest.mark.parametrize("given", [None, 1, 3])
def test_a_batch_without_rows_has_a_gradient(gpu, given):
    """An empty one: a training step without rows runs as any other."""
    announce(f"logprobs: no rows, {given} given")
    w = torch.randn(8, 50, device=gpu, requires_grad=True)
    hidden = torch.empty(0, 8, device=gpu)
    t = None if given is None else torch.empty((0,) if given == 1 else (0, given), dtype=torch.int64,
                                               device=gpu)
    r = call(hidden @ w, t, top_n=2, entropy=True)
    assert r.top_logprobs.requires_grad and not r.top_ids.requires_grad
    loss = r.entropy.sum() + r.top_logprobs.sum()
    if given is not None:
        assert r.logprobs.shape == t.shape
        loss = loss + r.logprobs.sum()
    loss.backward()
    assert w.grad.shape == w.shape and not w.grad.any()
    with torch.no_grad():
        r = call(hidden @ w, t, top_n=2, entropy=True)
    assert not r.entropy.requires_grad and r.top_ids.shape == (0, 2)
