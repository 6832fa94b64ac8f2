"""Continuing conversations over a shared paged cache, as measurable cases.

The operators, each in its plain form (elementary torch operations, 32 bits or more,
rounded once at the end) and as a program calls the framework's own:

  chunk    attention of each sequence's new tokens over its pages, causal inside the chunk
           (paged_attention_chunk_hip)
  rotary   rotary positions of q and k, half or interleaved layout, a whole head or part of
           it, frequencies scaled for long contexts, with or without the write of k and v
           into the cache's slots (rotary_embedding_hip, rotary_embedding_prefill_hip)
  fork     a sequence's rows of the block table are taken over by another sequence, the
           partly filled last page is copied (fork_pages_hip)
  move     whole pages move to other blocks, every table entry follows (move_pages_hip)

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
        # One user's draft tokens being verified: five tokens, launch latency.
        {"name": "chunk_verify_1", "kind": "chunk", "seqs": 1, "new_lo": 5, "new_hi": 5,
         "ctx_lo": 900, "ctx_hi": 900, "heads": 16, "kv_heads": 8, "block": 16},
        # A serving batch's draft tokens, long contexts: streaming the cache.
        {"name": "chunk_verify_48", "kind": "chunk", "seqs": 48, "new_lo": 4, "new_hi": 4,
         "ctx_lo": 1024, "ctx_hi": 8192, "heads": 32, "kv_heads": 8, "block": 16},
        # Next turns of several chats behind cached prefixes, ragged.
        {"name": "chunk_turns_12", "kind": "chunk", "seqs": 12, "new_lo": 20, "new_hi": 700,
         "ctx_lo": 0, "ctx_hi": 6000, "heads": 16, "kv_heads": 8, "block": 16},
        # One piece of a long prompt that is prefilled in pieces of about 512 tokens.
        {"name": "chunk_piece_509", "kind": "chunk", "seqs": 1, "new_lo": 509, "new_hi": 509,
         "ctx_lo": 12000, "ctx_hi": 12000, "heads": 32, "kv_heads": 8, "block": 32},
        # A question of 40 tokens about one very long document.
        {"name": "chunk_question_100k", "kind": "chunk", "seqs": 1, "new_lo": 40, "new_hi": 40,
         "ctx_lo": 100000, "ctx_hi": 100000, "heads": 32, "kv_heads": 8, "block": 16},
        # A large piece late in a long document: matrix products.
        {"name": "chunk_piece_2k_64k", "kind": "chunk", "seqs": 1, "new_lo": 2048, "new_hi": 2048,
         "ctx_lo": 64000, "ctx_hi": 64000, "heads": 32, "kv_heads": 8, "block": 16},
        # A long prompt's pieces at far positions, frequencies by parts, written to the cache.
        {"name": "rotary_write_8k", "kind": "rotary", "tokens": 8115, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "rotary_dim": 128, "layout": "half", "scaling": "yarn",
         "dtype": "bf16", "far": 131072, "write": True},
        # A quarter of each head, neighbouring pairs, in 32 bits.
        {"name": "rotary_part_fp32", "kind": "rotary", "tokens": 4093, "heads": 24, "kv_heads": 4,
         "head_dim": 128, "rotary_dim": 32, "layout": "interleaved", "scaling": "linear",
         "dtype": "fp32", "far": 1000000, "write": False},
        # One request sampled twice: its last page is copied, all layers.
        {"name": "fork_1", "kind": "fork", "forks": 1, "lo": 1000, "hi": 1000, "layers": 28,
         "kv_heads": 8, "block": 16, "blocks": 512},
        # A batch of 24 branches of eight running requests.
        {"name": "fork_24", "kind": "fork", "forks": 24, "lo": 100, "hi": 1000, "layers": 28,
         "kv_heads": 8, "block": 16, "blocks": 640},
        # A few pages of a model with eight layers, between two steps.
        {"name": "move_3", "kind": "move", "moves": 3, "rows": 16, "layers": 8, "kv_heads": 8,
         "block": 16, "blocks": 512},
        # A third of a fragmented cache moves together.
        {"name": "move_200", "kind": "move", "moves": 200, "rows": 64, "layers": 28,
         "kv_heads": 8, "block": 16, "blocks": 640},
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["chunk", "chunk", "chunk", "rotary", "rotary", "fork", "move"])
    if kind == "chunk":
        heads, kv_heads = rng.choice([(16, 8), (32, 8), (64, 8), (8, 8), (40, 8), (6, 2)])
        seqs = _log_int(rng, 1, 64)
        new = _log_int(rng, 1, min(4096, 16384 // seqs))
        # pages of the listed batch and the listed products at most
        far = int(min(300000 / seqs, 1.2e8 / (new * seqs) * 32 / heads, 100000))
        ctx = _log_int(rng, 1, max(2, far)) if rng.random() < 0.9 else 0
        return {"kind": kind, "seqs": seqs, "new_lo": max(1, int(new * rng.uniform(0.05, 1.0))),
                "new_hi": new, "ctx_lo": int(ctx * rng.uniform(0.0, 1.0)), "ctx_hi": ctx,
                "heads": heads, "kv_heads": kv_heads, "block": rng.choice([16, 16, 32, 64])}
    if kind == "rotary":
        head_dim, part = rng.choice([(128, 128), (128, 128), (128, 64), (128, 32), (64, 64),
                                     (80, 32), (256, 64), (192, 64)])
        heads, kv_heads = rng.choice([(16, 8), (32, 8), (24, 4), (8, 8), (5, 1)])
        write = head_dim == 128 and rng.random() < 0.4
        dtype = "bf16" if write else rng.choice(["bf16", "bf16", "fp16", "fp32"])
        size = (heads + kv_heads) * head_dim * (4 if dtype == "fp32" else 2)
        return {"kind": kind, "tokens": _log_int(rng, 1, min(16384, 80_000_000 // size)),
                "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "rotary_dim": part,
                "layout": rng.choice(["half", "half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "yarn", "llama3"]), "dtype": dtype,
                "far": _log_int(rng, 100, 2000000), "write": write}
    layers = rng.choice([28, 36, 8, 1])
    kv_heads, block = rng.choice([(8, 16), (8, 32), (4, 16), (2, 64)])
    page = layers * kv_heads * block * D * 2
    blocks = max(64, min(2048, 600_000_000 // page))
    if kind == "fork":
        hi = _log_int(rng, block, 30 * block)
        return {"kind": kind, "forks": _log_int(rng, 1, 32), "lo": max(1, hi // 4), "hi": hi,
                "layers": layers, "kv_heads": kv_heads, "block": block, "blocks": max(blocks, 320)}
    return {"kind": kind, "moves": _log_int(rng, 1, blocks // 3), "rows": _log_int(rng, 4, 256),
            "layers": layers, "kv_heads": kv_heads, "block": block, "blocks": blocks}


def _rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _chunk_lengths(case):
    """(new tokens, tokens already in the cache) of each sequence."""
    r = _rng(case)
    return [(r.randint(case["new_lo"], case["new_hi"]), r.randint(case["ctx_lo"], case["ctx_hi"]))
            for _ in range(case["seqs"])]


def _fork_plan(case):
    """Running requests' lengths, the source of each fork."""
    r = _rng(case)
    sources = max(1, min(8, case["forks"] // 3))
    lens = [r.randint(case["lo"], case["hi"]) for _ in range(sources)]
    return lens, [i % sources for i in range(case["forks"])]


def _move_plan(case):
    """Pages of each row of the table, the blocks that move and where to."""
    r = _rng(case)
    ids = list(range(case["blocks"]))
    r.shuffle(ids)
    src, dst, rest = (ids[:case["moves"]], ids[case["moves"]:2 * case["moves"]],
                      ids[2 * case["moves"]:])
    live = src + rest[:len(rest) // 2]
    r.shuffle(live)
    rows = [[] for _ in range(case["rows"])]
    for i, b in enumerate(live):
        rows[i % case["rows"]].append(b)
    return rows, src, dst


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape, std=1.0, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device=DEV).normal_(0.0, std, generator=g)


def _table(rows, width):
    t = torch.full((len(rows), max(width, 1)), -1, dtype=torch.int32)
    for i, r in enumerate(rows):
        t[i, :len(r)] = torch.tensor(r, dtype=torch.int32)
    return t.to(DEV)


# ---- frequencies ------------------------------------------------------------------

def _frequencies(case):
    """Angular frequencies in 64 bits and the factor on cos and sin."""
    d, base = case["rotary_dim"], 1e6
    inv = base ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    if case["scaling"] == "linear":
        return inv / 4.0, 1.0
    if case["scaling"] == "yarn":  # by parts: 4 times 32768 positions, 32 and 1 rotations
        turns = lambda n: d * math.log(32768 / (n * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(turns(32)), 0), min(math.ceil(turns(1)), d - 1)
        keep = 1 - ((torch.arange(d // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return inv * keep + inv / 4.0 * (1 - keep), 0.1 * math.log(4.0) + 1.0
    if case["scaling"] == "llama3":  # by wave length: 8 times 8192 positions
        turns = 8192 * inv / (2 * math.pi)
        smooth = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return inv * smooth + inv / 8.0 * (1 - smooth), 1.0
    return inv, 1.0


# ---- what a program has in hand before the call --------------------------------------

def _prepare_chunk(case, seed):
    lens, bs, hkv = _chunk_lengths(case), case["block"], case["kv_heads"]
    g = _gen(seed)
    pages = [(n + c + bs - 1) // bs for n, c in lens]
    blocks = sum(pages) + sum(pages) // 10 + 1
    perm = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), max(pages)), -1, dtype=torch.int32, device=DEV)
    cu, off = [0], 0
    for b, n in enumerate(pages):
        table[b, :n] = perm[off:off + n]
        off += n
        cu.append(cu[-1] + lens[b][0])
    kb, vb = (_randn(g, blocks, 2, hkv, bs, D) for _ in range(2))
    return {"kind": "chunk", "lens": lens, "block": bs, "k": kb[:, LAYER], "v": vb[:, LAYER],
            # normalised heads with learned weights: scores of a few units
            "q": _randn(g, cu[-1], case["heads"], D, std=2.0), "table": table,
            "seq_lens": torch.tensor([c for _, c in lens], dtype=torch.int32, device=DEV),
            "rows": torch.arange(len(lens), dtype=torch.int32, device=DEV),
            "cu": torch.tensor(cu, dtype=torch.int32, device=DEV), "most": max(n for n, _ in lens)}


def _prepare_rotary(case, seed):
    g, T, hq, hkv, d = (_gen(seed), case["tokens"], case["heads"], case["kv_heads"],
                        case["head_dim"])
    dtype = TYPES[case["dtype"]]
    qkv = _randn(g, T, (hq + 2 * hkv) * d, dtype=dtype)  # the fused projection's output
    inv, factor = _frequencies(case)
    s = {"kind": "rotary", "q": qkv[:, :hq * d].view(T, hq, d),
         "k": qkv[:, hq * d:(hq + hkv) * d].view(T, hkv, d),
         "v": qkv[:, (hq + hkv) * d:].view(T, hkv, d),
         "pos": torch.randint(0, case["far"], (T,), generator=g, device=DEV),
         "inv": inv.to(DEV), "factor": factor, "half": case["layout"] == "half",
         "write": case["write"]}
    if s["write"]:
        blocks = (T + 15) // 16 + 8
        order = torch.randperm(blocks, generator=g, device=DEV)
        t = torch.arange(T, device=DEV)
        s["slots"] = order[t // 16] * 16 + t % 16
        s["kb"], s["vb"] = (torch.zeros(blocks, 1, hkv, 16, d, dtype=dtype, device=DEV)
                            for _ in range(2))
    if own:
        from qwen3_engine_from_scratch_amd.kernels.rotary import Rotary
        s["rotary"] = Rotary(s["inv"], layout=case["layout"], attention_factor=factor)
    return s


def _pool(case, g):
    return [_randn(g, case["blocks"], case["layers"], case["kv_heads"], case["block"], D)
            for _ in range(2)]


def _prepare_fork(case, seed):
    lens, source = _fork_plan(case)
    bs, g = case["block"], _gen(seed)
    kb, vb = _pool(case, g)
    ids = torch.randperm(case["blocks"], generator=g, device=DEV).tolist()
    rows, at = [], 0
    for n in lens:
        p = (n + bs - 1) // bs
        rows.append(ids[at:at + p])
        at += p
    width = max(len(r) for r in rows) + 4
    table = _table(rows + [[] for _ in source], width)
    seq_lens = torch.zeros(table.shape[0], dtype=torch.int32, device=DEV)
    seq_lens[:len(lens)] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    return {"kind": "fork", "k": kb, "v": vb, "table": table, "seq_lens": seq_lens, "block": bs,
            "src": source, "dst": [len(lens) + i for i in range(len(source))],
            "tokens": [lens[i] for i in source], "new": ids[at:at + len(source)]}


def _prepare_move(case, seed):
    rows, src, dst = _move_plan(case)
    kb, vb = _pool(case, _gen(seed))
    return {"kind": "move", "k": kb, "v": vb, "src": src, "dst": dst,
            "table": _table(rows, max(len(r) for r in rows) + 4)}


def prepare(case, seed):
    return {"chunk": _prepare_chunk, "rotary": _prepare_rotary, "fork": _prepare_fork,
            "move": _prepare_move}[case["kind"]](case, seed)


# ---- one pass: the framework's operators ------------------------------------------------

def _own(s):
    if s["kind"] == "chunk":
        from qwen3_engine_from_scratch_amd.kernels.paged_attention import paged_attention_chunk_hip
        return paged_attention_chunk_hip(s["q"], s["k"], s["v"], s["table"], s["seq_lens"],
                                         s["rows"], s["cu"], s["block"], max_chunk=s["most"])
    if s["kind"] == "rotary":
        from qwen3_engine_from_scratch_amd.kernels.rotary import (rotary_embedding_hip,
                                                                  rotary_embedding_prefill_hip)
        if not s["write"]:
            return rotary_embedding_hip(s["q"], s["k"], s["pos"], s["rotary"])
        q, k = rotary_embedding_prefill_hip(s["q"], s["k"], s["v"], s["pos"], s["rotary"],
                                            s["slots"], s["kb"], s["vb"], 0)
        return q, k, s["kb"], s["vb"]
    if s["kind"] == "fork":
        from qwen3_engine_from_scratch_amd.kernels.paged_cache import fork_pages_hip
        fork_pages_hip(s["k"], s["v"], s["table"], s["seq_lens"], s["src"], s["dst"], s["tokens"],
                       s["new"])
        return s["k"], s["v"], s["table"], s["seq_lens"]
    from qwen3_engine_from_scratch_amd.kernels.paged_cache import move_pages_hip
    move_pages_hip(s["k"], s["v"], s["table"], s["src"], s["dst"])
    return s["k"], s["v"], s["table"]


# ---- one pass: the plain forms ------------------------------------------------------------

def _plain_chunk(s):
    q, bs = s["q"], s["block"]
    T, hq, _ = q.shape
    hkv = s["k"].shape[1]
    G = hq // hkv
    out = torch.empty_like(q)
    at = 0
    for b, (n, c) in enumerate(s["lens"]):
        L = n + c
        pages = s["table"][b, :(L + bs - 1) // bs].long()
        kc, vc = (x[pages].permute(1, 0, 2, 3).reshape(hkv, -1, D)[:, :L].float()
                  for x in (s["k"], s["v"]))
        kt = kc.transpose(1, 2).contiguous()
        step = max(1, int(2 ** 28 // (hq * L)))  # scores of at most 1 GB at once
        for i in range(0, n, step):
            m = min(step, n - i)
            qi = q[at + i:at + i + m].float().view(m, hkv, G, D).permute(1, 0, 2, 3)
            x = torch.matmul(qi.reshape(hkv, m * G, D), kt) * D ** -0.5
            keys = torch.arange(L, device=q.device)
            last = c + i + torch.arange(m, device=q.device).repeat_interleave(G)
            x.masked_fill_(keys[None, :] > last[:, None], float("-inf"))
            x = torch.exp(x - x.amax(-1, keepdim=True))
            o = torch.matmul(x, vc) / x.sum(-1, keepdim=True)
            out[at + i:at + i + m] = o.view(hkv, m, G, D).permute(1, 0, 2, 3).reshape(m, hq, D)
        at += n
    return out


def _plain_rotate(x, cos, sin, half):
    r = cos.shape[-1]
    a = x.float()
    cos, sin = cos[:, None], sin[:, None]
    if half:
        x1, x2 = a[..., :r], a[..., r:2 * r]
        y = torch.cat((x1 * cos - x2 * sin, x2 * cos + x1 * sin), -1)
    else:
        x1, x2 = a[..., 0:2 * r:2], a[..., 1:2 * r:2]
        y = torch.stack((x1 * cos - x2 * sin, x2 * cos + x1 * sin), -1).flatten(-2)
    return torch.cat((y.to(x.dtype), x[..., 2 * r:]), -1)


def _plain_rotary(s):
    angle = s["pos"].double()[:, None] * s["inv"]  # far positions need 64 bits
    cos, sin = ((f(angle) * s["factor"]).float() for f in (torch.cos, torch.sin))
    q, k = (_plain_rotate(s[x], cos, sin, s["half"]) for x in ("q", "k"))
    if not s["write"]:
        return q, k
    bs = s["kb"].shape[3]
    blk, off = s["slots"] // bs, s["slots"] % bs
    s["kb"][blk, 0, :, off] = k
    s["vb"][blk, 0, :, off] = s["v"]
    return q, k, s["kb"], s["vb"]


def _plain_fork(s):
    bs, table = s["block"], s["table"]
    dev = table.device
    src, dst, tok, new = (torch.tensor(s[x], device=dev) for x in ("src", "dst", "tokens", "new"))
    full, rest = tok // bs, tok % bs
    cols = torch.arange(table.shape[1], device=dev)
    rows = torch.where(cols < full[:, None], table[src], -1)
    part = rest > 0
    last = table[src[part], full[part]].long()
    rows[part, full[part]] = new[part].to(torch.int32)
    table[dst] = rows
    s["seq_lens"][dst] = tok.to(torch.int32)
    used = (torch.arange(bs, device=dev) < rest[part][:, None])[:, None, None, :, None]
    for x in (s["k"], s["v"]):
        x[new[part]] = torch.where(used, x[last], torch.zeros((), dtype=x.dtype, device=dev))
    return s["k"], s["v"], table, s["seq_lens"]


def _plain_move(s):
    table = s["table"]
    src, dst = (torch.tensor(s[x], device=table.device) for x in ("src", "dst"))
    for x in (s["k"], s["v"]):
        x[dst] = x[src]
    to = torch.arange(s["k"].shape[0], dtype=torch.int32, device=table.device)
    to[src] = dst.to(torch.int32)
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))
    return s["k"], s["v"], table


@torch.no_grad()
def run(s):
    if own:
        return _own(s)
    return {"chunk": _plain_chunk, "rotary": _plain_rotary, "fork": _plain_fork,
            "move": _plain_move}[s["kind"]](s)


# ---- what a pass cannot do without -----------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "chunk":
        lens, hq, hkv, bs = _chunk_lengths(case), case["heads"], case["kv_heads"], case["block"]
        keys = sum(n + c for n, c in lens)
        pages = sum((n + c + bs - 1) // bs for n, c in lens)
        return {"bytes": keys * hkv * D * 4 + sum(n for n, _ in lens) * hq * D * 4
                + 4 * pages + 12 * len(lens),
                "flops": 4 * D * hq * sum(n * c + n * (n + 1) // 2 for n, c in lens)}
    if kind == "rotary":
        T, hq, hkv, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
        size = 4 if case["dtype"] == "fp32" else 2
        n = 2 * (hq + hkv) * d * size + 8
        if case["write"]:  # v in, the cache's k and v out, the slot
            n += 3 * hkv * d * size + 8
        return {"bytes": T * n, "flops": T * (hq + hkv) * case["rotary_dim"] * 3}
    page = 2 * case["layers"] * case["kv_heads"] * case["block"] * D * 2  # K and V
    if kind == "fork":
        lens, source = _fork_plan(case)
        rest = [lens[i] % case["block"] for i in source]
        table = 8 * sum(lens[i] // case["block"] for i in source)
        return {"bytes": sum(page * r // case["block"] + page for r in rest if r) + table + 4,
                "flops": 0}
    rows, src, _ = _move_plan(case)
    return {"bytes": 2 * page * len(src) + 4 * case["rows"] * (max(len(r) for r in rows) + 4),
            "flops": 0}


# ---- the definitions in 64 bits -----------------------------------------------------------

def _exact_chunk(s):
    q, bs, table = s["q"].double(), s["block"], s["table"].cpu()
    hkv = s["k"].shape[1]
    G = q.shape[1] // hkv
    out = torch.empty_like(q)
    at = 0
    for b, (n, c) in enumerate(s["lens"]):
        for h in range(hkv):
            ks, vs = (torch.cat([x[int(p), h] for p in table[b, :-(-(n + c) // bs)]]).double()
                      for x in (s["k"], s["v"]))
            kt = ks.t().contiguous()
            for g in range(G):
                for i in range(0, n, 512):
                    e = min(n, i + 512)
                    L = c + e
                    x = torch.mm(q[at + i:at + e, h * G + g], kt[:, :L].contiguous()) / math.sqrt(D)
                    x += torch.full_like(x, float("-inf")).triu(c + i + 1)
                    w = torch.exp(x - torch.logsumexp(x, -1, keepdim=True))
                    out[at + i:at + e, h * G + g] = torch.mm(w, vs[:L])
        at += n
    return out


def _exact_rotary(case, s):
    # each pair as a complex number, turned by exp(i angle)
    turn = torch.polar(torch.full((), s["factor"], dtype=torch.float64, device=DEV).expand(
        len(s["pos"]), len(s["inv"])), s["pos"].double()[:, None] * s["inv"])[:, None]
    r, outs = case["rotary_dim"], []
    for x in (s["q"].double(), s["k"].double()):
        y = x.clone()
        p = x[..., :r]
        if s["half"]:
            z = torch.complex(p[..., :r // 2].contiguous(), p[..., r // 2:].contiguous()) * turn
            y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
        else:
            z = torch.view_as_complex(p.reshape(*p.shape[:-1], r // 2, 2).contiguous()) * turn
            y[..., :r] = torch.view_as_real(z).flatten(-2)
        outs.append(y)
    if not s["write"]:
        return tuple(outs)
    pools = []
    for new, old in ((outs[1], s["kb"]), (s["v"].double(), s["vb"])):
        flat = torch.zeros(old.shape[0] * old.shape[3], *new.shape[1:], dtype=torch.float64,
                           device=DEV)
        flat[s["slots"]] = new
        pools.append(flat.view(old.shape[0], old.shape[3], *new.shape[1:]).transpose(1, 2)[:, None])
    return (*outs, *pools)


def _exact_fork(s):
    k, v, table, lens, bs = s["k"], s["v"], s["table"].tolist(), s["seq_lens"].tolist(), s["block"]
    for a, b, n, new in zip(s["src"], s["dst"], s["tokens"], s["new"]):
        pages = [table[a][i] for i in range(n // bs)]
        if n % bs:
            for x in (k, v):
                x[new, :, :, :n % bs] = x[table[a][n // bs], :, :, :n % bs].clone()
                x[new, :, :, n % bs:] = 0
            pages.append(new)
        table[b] = pages + [-1] * (len(table[b]) - len(pages))
        lens[b] = n
    # copied bits, the values that they stand for: no arithmetic, so no 64-bit form of the pools
    return None, None, torch.tensor(table, dtype=torch.int32), torch.tensor(lens, dtype=torch.int32)


def _exact_move(s):
    to = dict(zip(s["src"], s["dst"]))
    table = [[to.get(b, b) for b in row] for row in s["table"].tolist()]
    return None, None, torch.tensor(table, dtype=torch.int32)


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "chunk":
        return _exact_chunk(s)
    if case["kind"] == "rotary":
        return _exact_rotary(case, s)
    return _exact_fork(s) if case["kind"] == "fork" else _exact_move(s)
