"""Many answers to one prompt, and how probable each is, as measurable cases.

The operators, each in its plain form (elementary torch operations, 32 bits or more,
rounded once at the end) and as a program calls the framework's own:

  shared    decode attention of a batch whose groups share a prefix of the paged cache: the
            prefix's pages serve all rows of a group at once
            (paged_attention_decode_shared_hip)
  logprobs  log probabilities of given tokens, the entropy of their distributions and the
            most likely tokens (token_logprobs)
  grad      the same as a training step uses it: log probabilities and entropies, and the
            gradient of the logits (token_logprobs and its backward pass)

Lengths and plans are part of a case (drawn from its own small generator), the tensors'
values come from the seed.
"""
import math
import random

import torch

own = False

D = 128          # head_dim of every attention here
DEV = "cuda"
LAYER = 1        # the layer of a two-layer pool that the attention cases read
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # One chat prompt answered four times: launch latency.
        {"name": "shared_4_900", "kind": "shared", "groups": 1, "group_lo": 4, "group_hi": 4,
         "alone": 0, "pre_lo": 896, "pre_hi": 896, "own_lo": 1, "own_hi": 40, "heads": 16,
         "kv_heads": 8, "block": 16},
        # Sixteen samples of one longer prompt, to be ranked.
        {"name": "shared_16_4k", "kind": "shared", "groups": 1, "group_lo": 16, "group_hi": 16,
         "alone": 0, "pre_lo": 4096, "pre_hi": 4096, "own_lo": 10, "own_hi": 600, "heads": 32,
         "kv_heads": 8, "block": 16},
        # A full serving batch behind one set of worked examples.
        {"name": "shared_64_8k", "kind": "shared", "groups": 1, "group_lo": 64, "group_hi": 64,
         "alone": 0, "pre_lo": 8192, "pre_hi": 8192, "own_lo": 1, "own_hi": 1000, "heads": 32,
         "kv_heads": 8, "block": 16},
        # Several prompts answered a few times each, beside requests that share nothing.
        {"name": "shared_groups_ragged", "kind": "shared", "groups": 6, "group_lo": 3,
         "group_hi": 12, "alone": 9, "pre_lo": 500, "pre_hi": 12000, "own_lo": 1, "own_hi": 900,
         "heads": 16, "kv_heads": 8, "block": 32},
        # Many conversations behind one system prompt: most keys are their own.
        {"name": "shared_256_2k", "kind": "shared", "groups": 1, "group_lo": 256,
         "group_hi": 256, "alone": 0, "pre_lo": 2000, "pre_hi": 2000, "own_lo": 50,
         "own_hi": 2500, "heads": 16, "kv_heads": 8, "block": 16},
        # Questions about one very long document.
        {"name": "shared_32_100k", "kind": "shared", "groups": 1, "group_lo": 32, "group_hi": 32,
         "alone": 0, "pre_lo": 100000, "pre_hi": 100000, "own_lo": 30, "own_hi": 400,
         "heads": 32, "kv_heads": 8, "block": 16},
        # One request's step, with its five most likely tokens: launch latency.
        {"name": "logprobs_step_1", "kind": "logprobs", "rows": 1, "vocab": 151936, "given": 1,
         "top": 5, "entropy": False, "temperature": 1.0, "dtype": "bf16", "masked": 0.0},
        # A serving batch's step, some rows held to a grammar (few tokens allowed).
        {"name": "logprobs_step_64", "kind": "logprobs", "rows": 64, "vocab": 151936, "given": 1,
         "top": 20, "entropy": True, "temperature": 1.0, "dtype": "bf16", "masked": 0.15},
        # Long prompts scored: streaming the logits.
        {"name": "logprobs_score_4k", "kind": "logprobs", "rows": 4096, "vocab": 151936,
         "given": 1, "top": 0, "entropy": True, "temperature": 1.0, "dtype": "bf16",
         "masked": 0.0},
        # Answers to choose from (four tokens a row) in 32 bits, an odd vocabulary.
        {"name": "logprobs_choices_fp32", "kind": "logprobs", "rows": 1003, "vocab": 50021,
         "given": 4, "top": 8, "entropy": False, "temperature": 0.7, "dtype": "fp32",
         "masked": 0.0},
        # A policy's training step on a few sequences.
        {"name": "grad_2k", "kind": "grad", "rows": 2048, "vocab": 151936, "given": 1, "top": 0,
         "entropy": True, "temperature": 1.0, "dtype": "bf16", "masked": 0.0},
        # One short answer, an odd vocabulary, 16 bits of the other kind.
        {"name": "grad_odd_fp16", "kind": "grad", "rows": 131, "vocab": 32003, "given": 1,
         "top": 0, "entropy": True, "temperature": 1.3, "dtype": "fp16", "masked": 0.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["shared", "shared", "shared", "logprobs", "logprobs", "grad"])
    if kind == "shared":
        heads, kv_heads = rng.choice([(16, 8), (32, 8), (64, 8), (8, 8), (40, 8), (6, 2)])
        groups = _log_int(rng, 1, 8)
        group = _log_int(rng, 2, 256 // groups)
        # keys of the listed document at most, and its products
        pre = _log_int(rng, 16, min(100000 // groups, 1.0e8 / (groups * group * heads)))
        own_hi = _log_int(rng, 1, max(2, min(8000, 200000 // (groups * group))))
        return {"kind": kind, "groups": groups, "group_lo": max(1, int(group * rng.uniform(0.2, 1.0))),
                "group_hi": group, "alone": rng.choice([0, 0, 1, 5, 20]),
                "pre_lo": max(1, int(pre * rng.uniform(0.1, 1.0))), "pre_hi": pre,
                "own_lo": max(1, int(own_hi * rng.uniform(0.0, 1.0))), "own_hi": own_hi,
                "heads": heads, "kv_heads": kv_heads, "block": rng.choice([16, 16, 32, 64])}
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    size = 4 if dtype == "fp32" else 2
    vocab = rng.choice([151936, _log_int(rng, 300, 152000), _log_int(rng, 300, 152000)])
    most = 1_240_000_000 if kind == "logprobs" else 620_000_000
    rows = _log_int(rng, 1, min(8192, most // (vocab * size)))
    return {"kind": kind, "rows": rows, "vocab": vocab, "given": rng.choice([1, 1, 2, 5]),
            "top": 0 if kind == "grad" or rows * vocab > 1.5e8 else rng.choice([0, 1, 5, 20, 50]),
            "entropy": kind == "grad" or rng.random() < 0.5,
            "temperature": rng.choice([1.0, 1.0, 0.6, 1.3]), "dtype": dtype,
            "masked": rng.choice([0.0, 0.0, 0.2])}


def _rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _plan(case):
    """For each group its shared tokens and its sequences' own tokens; what shares nothing
    is a group of one with no shared token."""
    r = _rng(case)
    plan = []
    for _ in range(case["groups"]):
        pre = r.randint(case["pre_lo"], case["pre_hi"])
        n = r.randint(case["group_lo"], case["group_hi"])
        # only whole pages are shared: a branch copies a page that is filled in part
        shared = pre - pre % case["block"]
        plan.append((shared, [pre - shared + r.randint(case["own_lo"], case["own_hi"])
                              for _ in range(n)]))
    for _ in range(case["alone"]):
        plan.append((0, [r.randint(case["own_lo"], max(case["own_hi"], case["pre_lo"]))]))
    r.shuffle(plan)
    return plan


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape, std=1.0, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device=DEV).normal_(0.0, std, generator=g)


# ---- what a program has in hand before the call --------------------------------------

def _prepare_shared(case, seed):
    plan, bs, hkv = _plan(case), case["block"], case["kv_heads"]
    g = _gen(seed)
    pages = [s // bs + sum(-(-n // bs) for n in ns) for s, ns in plan]
    blocks = sum(pages) + sum(pages) // 10 + 1
    perm = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)
    B = sum(len(ns) for _, ns in plan)
    table = torch.full((B, max(s // bs + max(-(-n // bs) for n in ns) for s, ns in plan)), -1,
                       dtype=torch.int32, device=DEV)
    at, b, cu, lens = 0, 0, [0], []
    for s, ns in plan:
        pre = perm[at:at + s // bs]
        at += s // bs
        for n in ns:
            p = -(-n // bs)
            table[b, :s // bs] = pre
            table[b, s // bs:s // bs + p] = perm[at:at + p]
            at += p
            lens.append(s + n)
            b += 1
        cu.append(b)
    kb, vb = (_randn(g, blocks, 2, hkv, bs, D) for _ in range(2))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return {"kind": "shared", "plan": plan, "lens": lens, "block": bs, "k": kb[:, LAYER],
            "v": vb[:, LAYER], "table": table,
            # normalised heads with learned weights: scores of a few units
            "q": _randn(g, B, case["heads"], D, std=2.0),
            "seq_lens": i32([n - 1 for n in lens]),  # before the step's token
            "rows": torch.arange(B, dtype=torch.int32, device=DEV),
            "cu": i32(cu), "shared": i32([s for s, _ in plan])}


def _prepare_logits(case, seed):
    g, T, V = _gen(seed), case["rows"], case["vocab"]
    logits = torch.empty(T, V, dtype=TYPES[case["dtype"]], device=DEV)
    tokens = torch.empty(T, case["given"], dtype=torch.int64, device=DEV)
    step = max(1, (1 << 27) // V)
    for i in range(0, T, step):
        x = torch.empty(min(step, T - i), V, device=DEV).normal_(0.0, 2.5, generator=g)
        if case["masked"]:  # a grammar allows a dozen tokens of these rows
            held = torch.rand(len(x), generator=g, device=DEV) < case["masked"]
            allowed = torch.randint(0, V, (len(x), 12), generator=g, device=DEV)
            keep = torch.zeros_like(x, dtype=torch.bool).scatter_(1, allowed, True)
            x.masked_fill_(held[:, None] & ~keep, float("-inf"))
        logits[i:i + step] = x
        for k in range(case["given"]):  # drawn from the distribution
            noise = -torch.log(torch.empty_like(x).exponential_(generator=g))
            tokens[i:i + step, k] = (x + noise).argmax(1)
    s = {"kind": case["kind"], "logits": logits, "top": case["top"], "entropy": case["entropy"],
         "tokens": tokens[:, 0].contiguous() if case["given"] == 1 else tokens,
         "temperature": case["temperature"]}
    if case["kind"] == "grad":
        # advantages, an entropy bonus, both over the number of tokens
        s["g"] = torch.empty(s["tokens"].shape, device=DEV).normal_(0.0, 1.0, generator=g)
        s["g_entropy"] = torch.full((T,), -0.01, device=DEV)
        s["leaf"] = logits.requires_grad_(True)
    return s


def prepare(case, seed):
    return (_prepare_shared if case["kind"] == "shared" else _prepare_logits)(case, seed)


# ---- one pass: the framework's operators ------------------------------------------------

def _own(s):
    if s["kind"] == "shared":
        from qwen3_engine_from_scratch_amd.kernels.paged_attention import \
            paged_attention_decode_shared_hip
        return paged_attention_decode_shared_hip(s["q"], s["k"], s["v"], s["table"],
                                                 s["seq_lens"], s["rows"], s["cu"], s["shared"],
                                                 s["block"])
    from qwen3_engine_from_scratch_amd.sampling import token_logprobs
    if s["kind"] == "logprobs":
        with torch.no_grad():
            r = token_logprobs(s["logits"], s["tokens"], top_n=s["top"], entropy=s["entropy"],
                               temperature=s["temperature"])
        return {k: v for k, v in r._asdict().items() if v is not None}
    r = token_logprobs(s["leaf"], s["tokens"], entropy=True, temperature=s["temperature"])
    grad, = torch.autograd.grad([r.logprobs, r.entropy], [s["leaf"]], [s["g"], s["g_entropy"]])
    return {"logprobs": r.logprobs.detach(), "entropy": r.entropy.detach(), "grad": grad}


# ---- one pass: the plain forms ------------------------------------------------------------

def _gather(x, pages, hkv):
    return x[pages.long()].permute(1, 0, 2, 3).reshape(hkv, -1, D).float()


def _attend(q, k, v):
    """Running form of attention over some keys: maximum, sum and weighted sum."""
    x = torch.matmul(q, k.transpose(1, 2).contiguous()) * D ** -0.5
    m = x.amax(-1, keepdim=True)
    x = torch.exp(x - m)
    return m, x.sum(-1, keepdim=True), torch.matmul(x, v)


def _plain_shared(s):
    q, bs = s["q"], s["block"]
    hq, hkv = q.shape[1], s["k"].shape[1]
    G = hq // hkv
    out = torch.empty_like(q)
    b = 0
    for shared, ns in s["plan"]:
        n, p = len(ns), shared // bs
        qg = q[b:b + n].float().view(n, hkv, G, D).transpose(0, 1)
        if shared:  # all rows of the group against the prefix, once
            pre = _attend(qg.reshape(hkv, n * G, D), *(_gather(x, s["table"][b, :p], hkv)
                                                       for x in (s["k"], s["v"])))
            pre = [x.view(hkv, n, G, -1) for x in pre]
        for i, own_n in enumerate(ns):
            pages = s["table"][b + i, p:p + -(-own_n // bs)]
            m, l, o = _attend(qg[:, i], *(_gather(x, pages, hkv)[:, :own_n]
                                          for x in (s["k"], s["v"])))
            if shared:
                pm, pl, po = (x[:, i] for x in pre)
                top = torch.maximum(m, pm)
                a, c = torch.exp(m - top), torch.exp(pm - top)
                l, o = l * a + pl * c, o * a + po * c
            out[b + i] = (o / l).reshape(hq, D)
        b += n
    return out


def _plain_logprobs(s, grads=False):
    logits, tokens, n = s["logits"].detach(), s["tokens"], s["top"]
    T, V = logits.shape
    lp, ent, ids, tops, dx = [], [], [], [], []
    step = max(1, (1 << 27) // V)
    for i in range(0, T, step):
        x = logits[i:i + step].float()
        if n:
            order = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :n]
        z = x / s["temperature"]
        z = z - z.amax(1, keepdim=True)
        e = torch.exp(z)
        total = e.sum(1, keepdim=True)
        z = z - torch.log(total)  # log probabilities
        t = tokens[i:i + step].view(len(z), -1)
        lp.append(z.gather(1, t).view(tokens[i:i + step].shape))
        if n:
            ids.append(order)
            tops.append(z.gather(1, order))
        if s["entropy"]:
            p = e / total
            h = -torch.where(p > 0, p * z, 0.0).sum(1)
            ent.append(h)
        if grads:
            g = s["g"][i:i + step].view(len(z), -1)
            gh = s["g_entropy"][i:i + step, None]
            d = -p * (g.sum(1, keepdim=True) + torch.where(p > 0, gh * (z + h[:, None]), 0.0))
            d.scatter_add_(1, t, g)
            dx.append((d / s["temperature"]).to(logits.dtype))
    r = {"logprobs": torch.cat(lp)}
    if s["entropy"]:
        r["entropy"] = torch.cat(ent)
    if n:
        r["top_ids"], r["top_logprobs"] = torch.cat(ids), torch.cat(tops)
    if grads:
        r["grad"] = torch.cat(dx)
    return r


def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return _plain_shared(s) if s["kind"] == "shared" else _plain_logprobs(s, s["kind"] == "grad")


# ---- what a pass cannot do without -----------------------------------------------------

def work(case):
    if case["kind"] == "shared":
        plan, hq, hkv, bs = _plan(case), case["heads"], case["kv_heads"], case["block"]
        B = sum(len(ns) for _, ns in plan)
        keys = sum(s + sum(ns) for s, ns in plan)
        pages = sum(s // bs + sum(-(-n // bs) for n in ns) for s, ns in plan)
        return {"bytes": keys * hkv * D * 4 + B * hq * D * 4 + 4 * pages + 8 * B + 8 * len(plan),
                "flops": 4 * D * hq * sum(s * len(ns) + sum(ns) for s, ns in plan)}
    T, V = case["rows"], case["vocab"]
    size = 4 if case["dtype"] == "fp32" else 2
    small = T * (case["given"] * 12 + (4 if case["entropy"] else 0) + 12 * case["top"])
    if case["kind"] == "logprobs":
        return {"bytes": T * V * size + small, "flops": 6 * T * V}
    return {"bytes": 2 * T * V * size + small + 8 * T, "flops": 12 * T * V}


# ---- the definitions in 64 bits -----------------------------------------------------------

def _exact_shared(s):
    q, bs, table = s["q"].double(), s["block"], s["table"].cpu()
    hkv = s["k"].shape[1]
    G = q.shape[1] // hkv
    out = torch.empty_like(q)
    for b, L in enumerate(s["lens"]):
        at = table[b, :-(-L // bs)].to(DEV).long()
        k, v = (x.index_select(0, at).transpose(0, 1).flatten(1, 2)[:, :L] for x in (s["k"], s["v"]))
        for h in range(hkv):
            w = torch.mm(k[h].double(), q[b, h * G:(h + 1) * G].t().contiguous()) / math.sqrt(D)
            w = torch.exp(w - torch.logsumexp(w, 0, keepdim=True))
            out[b, h * G:(h + 1) * G] = torch.mm(w.t().contiguous(), v[h].double())
    return out


def _exact_logprobs(s, grads=False):
    logits, tokens = s["logits"].detach(), s["tokens"]
    T, V = logits.shape
    r = {"logprobs": torch.empty(tokens.shape, dtype=torch.float64, device=DEV)}
    if s["entropy"]:
        r["entropy"] = torch.empty(T, dtype=torch.float64, device=DEV)
    if s["top"]:
        r["top_ids"] = torch.empty(T, s["top"], dtype=torch.int64, device=DEV)
        r["top_logprobs"] = torch.empty(T, s["top"], dtype=torch.float64, device=DEV)
    if grads:
        r["grad"] = torch.empty(T, V, dtype=torch.float64, device=DEV)
    step = max(1, (1 << 26) // V)
    for i in range(0, T, step):
        e = min(T, i + step)
        z = logits[i:e].double() / s["temperature"]
        lse = torch.logsumexp(z, 1, keepdim=True)
        t = tokens[i:e].reshape(e - i, -1)
        r["logprobs"][i:e] = (torch.gather(z, 1, t) - lse).view(tokens[i:e].shape)
        if s["top"]:
            # the value first, the index among equals: one key of both
            rank = torch.argsort(-logits[i:e].double(), dim=1, stable=True)[:, :s["top"]]
            r["top_ids"][i:e] = rank
            r["top_logprobs"][i:e] = torch.gather(z, 1, rank) - lse
        if s["entropy"]:
            p = torch.softmax(z, 1)
            mean = (p * z.nan_to_num(neginf=0.0)).sum(1)
            r["entropy"][i:e] = lse[:, 0] - mean
        if grads:
            # d lp_t / d z = one(t) - p;  d H / d z = p (mean z - z)
            d = p * ((mean[:, None] - z) * s["g_entropy"][i:e, None].double()).nan_to_num(
                posinf=0.0, neginf=0.0)
            for k in range(t.shape[1]):
                g = s["g"][i:e].reshape(e - i, -1)[:, k, None].double()
                d -= g * p
                d.scatter_add_(1, t[:, k, None], g)
            r["grad"][i:e] = d / s["temperature"]
    return r


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "shared":
        return _exact_shared(s)
    return _exact_logprobs(s, case["kind"] == "grad")
