"""token_logprobs refuses bad calls before anything is launched (CPU), and its oracle is
pinned to torch's own functions."""
import pytest
import torch

from oracle.logprobs import Rows, ranking
from qwen3_engine_from_scratch_amd import _lib
from qwen3_engine_from_scratch_amd.sampling import token_logprobs

FAKE = 1 << 20  # 16-byte aligned, never dereferenced on these paths


def test_oracle_is_log_softmax():
    x = torch.randn(4, 50, dtype=torch.float64, requires_grad=True)
    r = Rows(x.detach(), 0.7)
    lp = torch.log_softmax(x / 0.7, 1)
    assert (r.logp - lp).abs().max() < 1e-12
    ent = -(lp.exp() * lp).sum(1)
    assert (r.entropy - ent).abs().max() < 1e-12
    t = torch.tensor([[1, 1], [3, 4], [0, 49], [7, 8]])
    g, ge = torch.randn(4, 2, dtype=torch.float64), torch.randn(4, dtype=torch.float64)
    ids = ranking(x.detach(), 3)
    h = torch.randn(4, 3, dtype=torch.float64)
    loss = (lp.gather(1, t) * g).sum() + (lp.gather(1, ids) * h).sum() + (ent * ge).sum()
    want, = torch.autograd.grad(loss, x)
    got, off = r.gradient(t, g, ids, h, ge)
    assert (got - want).abs().max() < 1e-12 and (off > 0).all()


def test_oracle_ranking():
    x = torch.tensor([[1.0, float("nan"), 2.0, 2.0, -0.0, 0.0, float("inf"), float("-inf")]])
    assert ranking(x, 8).tolist() == [[1, 6, 2, 3, 0, 4, 5, 7]]


def _call(**over):
    a = dict(x=FAKE, st=100, dt=0, rows=4, vocab=100, tok=FAKE, given=1, temp=1.0, lp=FAKE,
             ent=None, top=0, ids=None, tlp=None, stats=None, ws=FAKE, wsb=1 << 30)
    a.update(over)
    return _lib.load().qwen3_token_logprobs(
        a["x"], a["st"], a["dt"], a["rows"], a["vocab"], a["tok"], a["given"], a["temp"], a["lp"],
        a["ent"], a["top"], a["ids"], a["tlp"], a["stats"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("code,over", [
    (-1, dict(x=None)), (-1, dict(tok=None)), (-1, dict(lp=None)), (-1, dict(top=3)),
    (-1, dict(top=3, ids=FAKE)), (-1, dict(rows=-1)), (-1, dict(vocab=0)), (-1, dict(st=99)),
    (-1, dict(vocab=(1 << 30) + 1, st=1 << 31)), (-1, dict(temp=0.0)), (-1, dict(temp=-1.0)),
    (-1, dict(temp=float("nan"))), (-1, dict(temp=float("inf"))), (-1, dict(temp=1e-39)),
    (-3, dict(dt=3)), (-3, dict(dt=-1)), (-3, dict(given=65)), (-3, dict(given=-1)),
    (-3, dict(top=65, ids=FAKE, tlp=FAKE)), (-3, dict(top=101, ids=FAKE, tlp=FAKE)),
    (-2, dict(x=FAKE + 1)), (-2, dict(dt=2, x=FAKE + 2)),
    (-4, dict(vocab=100000, st=100000, ws=None)), (-4, dict(vocab=100000, st=100000, wsb=16)),
    (-2, dict(vocab=100000, st=100000, ws=FAKE + 8)), (-1, dict(rows=1 << 33)),
])
def test_refuses(code, over):
    assert _call(**over) == code, _lib.load().qwen3_attn_last_error()


def _grad(**over):
    a = dict(x=FAKE, st=100, dt=0, rows=4, vocab=100, tok=FAKE, given=1, temp=1.0, ent=FAKE, top=0,
             ids=None, stats=FAKE, g=FAKE, ge=FAKE, gt=None, dx=FAKE, dst=100)
    a.update(over)
    return _lib.load().qwen3_token_logprobs_grad(
        a["x"], a["st"], a["dt"], a["rows"], a["vocab"], a["tok"], a["given"], a["temp"], a["ent"],
        a["top"], a["ids"], a["stats"], a["g"], a["ge"], a["gt"], a["dx"], a["dst"], None)


@pytest.mark.parametrize("code,over", [
    (-1, dict(x=None)), (-1, dict(stats=None)), (-1, dict(dx=None)), (-1, dict(tok=None)),
    (-1, dict(ent=None)), (-1, dict(gt=FAKE)), (-1, dict(dst=99)), (-1, dict(temp=0.0)),
    (-2, dict(dx=FAKE + 1)), (-3, dict(dt=7)), (-1, dict(rows=1 << 33)),
])
def test_gradient_refuses(code, over):
    assert _grad(**over) == code, _lib.load().qwen3_attn_last_error()


def test_nothing_to_do_is_no_error():
    assert _call(rows=0) == 0 and _grad(rows=0) == 0


def test_workspace_bytes():
    f = _lib.load().qwen3_token_logprobs_workspace_bytes
    assert f(1, 151936, 0, 5) > 0 and f(4096, 151936, 0, 5) == 0 and f(1, 100, 0, 5) == 0
    for bad in ((0, 100, 0, 5), (1, 0, 0, 5), (1, 100, 3, 5), (1, 100, 0, 65), (1, 100, 0, -1)):
        assert f(*bad) == 0


def test_wrapper_refuses():
    x = torch.zeros(4, 100, dtype=torch.bfloat16)
    t = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        token_logprobs(x, t)
    for args, kw in (((x[0], t), {}), ((x.to(torch.float64), t), {}), ((x.t(), None), dict(top_n=1)),
                     ((x, t.int()), {}), ((x, t[:3]), {}), ((x, t[:, None, None]), {}),
                     ((x, torch.zeros(4, 65, dtype=torch.int64)), {}),
                     ((x, torch.zeros(4, 0, dtype=torch.int64)), {}), ((x, t), dict(top_n=-1)),
                     ((x, t), dict(top_n=65)), ((x[:, :3], t), dict(top_n=4)),
                     ((x, t), dict(temperature=0.0)), ((x, t), dict(temperature=float("nan"))),
                     ((x, None), {}), ((x[:, :0], t), {}), ((x[:1].expand(4, 100), t), {})):
        with pytest.raises(ValueError):
            token_logprobs(*args, **kw)


def test_forward_mode_is_refused():
    """A dual tensor needs no gradient and has a data pointer: its tangent would be lost."""
    x, t = torch.zeros(4, 100), torch.zeros(4, dtype=torch.int64)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for logits in (dual, dual[1:3]):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                token_logprobs(logits, t[:len(logits)])
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            token_logprobs(x, t)  # (one without a tangent is not meant)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda z: token_logprobs(z, t).logprobs, (x,), (x,))
