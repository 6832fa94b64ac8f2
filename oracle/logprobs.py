"""Log probabilities, entropies, ranking and the logits' gradient from their definitions
in 64 bits, with what a computation in 32 bits may be off."""
import torch

EPS = 2.0 ** -23


def ranking(logits, n):
    """The n largest logits of each row: NaN first, then falling, the lower index first
    among equal ones (-0 is 0)."""
    x = logits.double() + 0.0
    x = torch.where(torch.isnan(x), torch.full_like(x, float("inf")), x)
    nan = torch.isnan(logits)
    out = torch.empty(logits.shape[0], n, dtype=torch.int64)
    for r in range(logits.shape[0]):
        first = torch.nonzero(nan[r])[:, 0]
        rest = torch.nonzero(~nan[r])[:, 0]
        order = rest[torch.sort(x[r][rest], descending=True, stable=True)[1]]
        out[r] = torch.cat([first, order])[:n]
    return out


class Rows:
    """A batch of rows: z = logits / temperature, log p, p, entropy and the bounds below."""

    def __init__(self, logits, temperature=1.0):
        z = logits.double() / temperature
        top = z.amax(1, keepdim=True)
        z = z - top
        e = torch.exp(z)
        s = e.sum(1, keepdim=True)
        self.logp = z - torch.log(s)
        self.logp[self.logp < -torch.finfo(torch.float32).max] = -float("inf")  # in 32 bits
        self.p = e / s
        self.temperature = temperature
        gone = self.p == 0
        terms = torch.where(gone, torch.zeros_like(z), self.p * self.logp)
        self.entropy = -terms.sum(1)
        # |y|, y = log2 of a term over the largest, as the sums' exponents are rounded
        y = torch.where(gone, torch.zeros_like(z), z.abs() / 0.6931471805599453)
        self.y1, self.y2 = (self.p * y).sum(1), (self.p * y * y).sum(1)
        self.depth = 40 + logits.shape[1] / 8192  # additions on the way of any term

    def sum_error(self):
        """Of log s: each term off by EPS (1 + |y|) (exponent: a multiply-add and the
        factor's rounding; the exponential: one unit), each addition by EPS / 2."""
        return EPS * (self.y1 + 1 + self.depth / 2)

    def logprob_error(self, logp):
        """logp = ln 2 (y - log2 s): y off by EPS |y| (|y| ln 2 <= |logp| + log s), the
        logarithm and the two last roundings by EPS of what they give."""
        log_s = -self.logp.amax(1)
        return self.sum_error()[:, None] + EPS * (3 * logp.abs() + 3 * log_s[:, None])

    def entropy_error(self):
        """H = ln 2 (log2 s - s1 / s), s1 = sum e y: its terms off as those of s, times |y|."""
        return (self.sum_error() * (1 + 2 * self.y1) + EPS * (self.y2 + self.y1)
                + 3 * EPS * (self.entropy.abs() + self.y1))

    def gradient(self, tokens=None, g=None, ids=None, h=None, g_entropy=None):
        """d sum(g logp[tokens] + h logp[ids] + g_entropy entropy) / d logits and its bound
        before the rounding to the logits' type."""
        n, V = self.p.shape
        one = torch.zeros(n, V, dtype=torch.float64)
        mass = torch.zeros(n, 1, dtype=torch.float64)
        size = torch.zeros(n, 1, dtype=torch.float64)
        for t, w in ((tokens, g), (ids, h)):
            if w is None:
                continue
            t, w = t.reshape(n, -1), w.double().reshape(n, -1)
            ok = (t >= 0) & (t < V)
            w = torch.where(ok, w, torch.zeros_like(w))
            one.scatter_add_(1, t.clamp(0, V - 1), w)
            mass += w.sum(1, keepdim=True)
            size += w.abs().sum(1, keepdim=True)
        gh = torch.zeros(n, 1, dtype=torch.float64) if g_entropy is None else g_entropy.double()[:, None]
        lp = torch.where(self.p == 0, torch.zeros_like(self.logp), self.logp)
        ent = self.entropy[:, None]
        d = one - self.p * (mass + gh * (lp + ent))
        # p off by EPS (1 + |log2 p| and the sum's), the bracket by its parts' errors
        rel = EPS * (3 + 2 * lp.abs()) + self.sum_error()[:, None] + 3 * EPS * (-self.logp.amax(1))[:, None]
        off = self.p * ((size + gh.abs() * (lp.abs() + ent.abs())) * (rel + 4 * EPS)
                        + size * 130 * EPS
                        + gh.abs() * (self.logprob_error(lp) + self.entropy_error()[:, None]))
        off = off + 4 * EPS * one.abs() + 130 * EPS * torch.where(one != 0, size, torch.zeros_like(one))
        return d / self.temperature, off / self.temperature
