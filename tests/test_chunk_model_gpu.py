"""The new operators together, as a program uses them: prompts prefilled in pieces,
requests behind a shared prefix, draft tokens verified and taken back, the pool
compacted under running requests -- against the fp32 oracle of the whole sequence
(the bar of test_model_gpu.py) and against the same steps without them."""
import pytest
import torch

from conftest import announce
from oracle import model as om
from test_model_gpu import _pool, _rel, _tiny

pytestmark = pytest.mark.gpu


def _check_logits(got, state, cfg, seq, at, what):
    """got: logits of positions `at` of seq.  Bar: no further from fp32 than twice the
    reference's own bf16 forward, or 0.03."""
    ref = om.qwen3_logits_ref(state, cfg, seq)[at]
    ref16 = om.qwen3_logits_ref(state, cfg, seq, dtype=torch.bfloat16)[at]
    e, e16 = _rel(got, ref), _rel(ref16, ref)
    announce(f"  {what}: rel err {e:.4f} (reference bf16 forward: {e16:.4f})")
    assert e <= max(2 * e16, 0.03), (what, e, e16)


def test_extend_in_pieces(gpu):
    from qwen3_engine_from_scratch_amd.PagedKVcache import PagedKVCache

    model, state, cfg = _tiny(seed=1)
    model = model.to(gpu)
    g = torch.Generator().manual_seed(3)
    seqs = [torch.randint(0, cfg.vocab_size, (n,), generator=g) for n in (150, 40, 97)]
    pieces = [[64, 64, 22], [1, 38, 1], [0, 96, 1]]
    announce("extend: three prompts in pieces of their own")
    pool = _pool(cfg, gpu)
    caches = [PagedKVCache(pool) for _ in seqs]
    got = [[] for _ in seqs]
    for step in range(3):
        lens = [p[step] for p in pieces]
        ids = torch.zeros(3, max(lens), dtype=torch.long)
        for i, (s, n) in enumerate(zip(seqs, lens)):
            ids[i, :n] = s[sum(pieces[i][:step]):][:n]
        out = model.extend(ids.to(gpu), caches, lens).cpu()
        for i, n in enumerate(lens):
            got[i].append(out[i, :n])
            assert not out[i, n:].any()
    for i, s in enumerate(seqs):
        assert caches[i].seq_len == len(s) and int(pool.seq_lens[caches[i].row_id]) == len(s)
        _check_logits(torch.cat(got[i]), state, cfg, s, slice(None), f"prompt {i}")
    assert not model.extend(torch.zeros(3, 2, dtype=torch.long, device=gpu), caches, [0, 0, 0]).any()


def test_forks_draft_tokens_and_compaction(gpu):
    from qwen3_engine_from_scratch_amd.PagedKVcache import PagedKVCache, fork_caches

    model, state, cfg = _tiny(seed=2)
    model = model.to(gpu)
    g = torch.Generator().manual_seed(5)
    base = torch.randint(0, cfg.vocab_size, (75,), generator=g)
    tails = [torch.randint(0, cfg.vocab_size, (n,), generator=g) for n in (20, 7, 33)]
    announce("one prompt forked, tails appended, drafts verified, pool compacted, decode")
    pool = _pool(cfg, gpu, blocks=48)
    lost = PagedKVCache(pool)
    root = PagedKVCache(pool)
    model.extend(torch.randint(0, cfg.vocab_size, (1, 60), generator=g).to(gpu), lost)
    model.extend(base[None].to(gpu), root)
    kids = fork_caches([root] * 3, [75, 64, 70])
    seqs = [torch.cat((base[:n], t)) for n, t in zip((75, 64, 70), tails)]
    ids = torch.zeros(3, 33, dtype=torch.long)
    for i, t in enumerate(tails):
        ids[i, :len(t)] = t
    out = model.extend(ids.to(gpu), kids, [len(t) for t in tails]).cpu()
    for i, (s, t) in enumerate(zip(seqs, tails)):
        _check_logits(out[i, :len(t)], state, cfg, s, slice(len(s) - len(t), None), f"branch {i}")
    # four draft tokens each, of which two are kept; one branch gives back into the prefix
    drafts = torch.randint(0, cfg.vocab_size, (3, 4), generator=g)
    out = model.extend(drafts.to(gpu), kids).cpu()
    for i in range(3):
        seqs[i] = torch.cat((seqs[i], drafts[i]))
        _check_logits(out[i], state, cfg, seqs[i], slice(-4, None), f"drafts {i}")
        kids[i].truncate(len(seqs[i]) - 2)
        seqs[i] = seqs[i][:-2]
    kids[1].truncate(20)
    seqs[1] = seqs[1][:20]
    lost.free()
    root.free()
    assert pool.compact(kids) > 0
    more = torch.randint(0, cfg.vocab_size, (3, 3), generator=g)
    for step in range(3):
        out = model(more[:, step:step + 1].to(gpu), kv_cache=kids).cpu()
        for i in range(3):
            seqs[i] = torch.cat((seqs[i], more[i, step:step + 1]))
            _check_logits(out[i], state, cfg, seqs[i], slice(-1, None), f"decode {i}.{step}")
    for k in kids:
        k.free()
    assert sorted(pool.free_block_ids) == list(range(48)) and not pool._extra_holders


@pytest.mark.parametrize("use_graph", [False, True])
def test_engine_prefix_and_pieces(gpu, use_graph):
    """Every token near the oracle's choice given the tokens before it, with and
    without shared prefixes and pieces (0.15 of that step's greatest logit, as
    test_model_gpu.py)."""
    from qwen3_engine_from_scratch_amd.engine import Engine, GenRequest

    model, state, cfg = _tiny(seed=3)
    model = model.to(gpu)
    g = torch.Generator().manual_seed(9)
    system = torch.randint(0, cfg.vocab_size, (53,), generator=g).tolist()
    asks = [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in (5, 40, 1, 18)]
    pool = _pool(cfg, gpu, blocks=96, max_requests=24)
    announce(f"engine with a shared prefix, pieces of 16 tokens, graph={use_graph}")
    engine = Engine(model, pool, max_batch=4, use_graph=use_graph, prefill_chunk=16)
    prefix = engine.cache_prefix(system)
    assert prefix.seq_len == 53
    reqs = [GenRequest(i, a, 6, prefix=prefix) for i, a in enumerate(asks)]
    reqs.append(GenRequest(4, system + asks[1], 6))
    reqs.append(GenRequest(5, asks[3][:9], 6))
    engine.generate(reqs)
    free = pool.free_count
    prefix.free()
    assert pool.free_count == free + 4 and not pool._extra_holders
    for r in reqs:
        prompt = (system if r.prefix is not None else []) + r.prompt
        assert len(r.output_ids) == 6
        ref = om.qwen3_logits_ref(state, cfg, torch.tensor(prompt + r.output_ids))
        for k, tok in enumerate(r.output_ids):
            row = ref[len(prompt) - 1 + k]
            assert row[tok] >= row.max() - 0.15, (r.request_id, k)
    engine.close()


def test_scaled_rope_tables_follow_the_rotary_operator(gpu):
    """The model's tables with rope_scaling hold the angles and the factor that the
    rotary operator turns by: the fused QK-norm step's rotation of a normalised head
    against it, both rounded to bf16 at most three times (cos, product, sum: each half a
    step of values up to the factor)."""
    from qwen3_engine_from_scratch_amd.kernels.pre_attention import qk_norm_rope_prefill, rope_tables
    from qwen3_engine_from_scratch_amd.kernels.rotary import make_rotary, rotary_embedding_hip

    announce("scaled tables against the rotary operator")
    scaling = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}
    cos, sin = rope_tables(128, 1e6, 16384, device=gpu, scaling=scaling)
    rot = make_rotary(128, 1e6, scaling=scaling, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(1)
    q = torch.randn(50, 4, 128, generator=g, device=gpu).to(torch.bfloat16)
    k = torch.randn(50, 2, 128, generator=g, device=gpu).to(torch.bfloat16)
    w = torch.ones(128, dtype=torch.bfloat16, device=gpu)
    pos = torch.randint(0, 16384, (50,), generator=g, device=gpu)
    kb = torch.zeros(1, 1, 2, 16, 128, dtype=torch.bfloat16, device=gpu)
    qf, kf = qk_norm_rope_prefill(q, k, k, w, w, 1e-6, cos, sin, pos, None, kb, kb.clone(), 0)

    def norm(x):
        y = x.float()
        return (y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + 1e-6)).to(torch.bfloat16)

    qn, kn = norm(q), norm(k)
    qr, kr = rotary_embedding_hip(qn, kn, pos, rot)
    for a, b, x in ((qf, qr, qn), (kf, kr, kn)):
        size = (x.float().abs() + x.float().abs().roll(64, -1)) * rot.attention_factor
        # cos, product and sum rounded here, the sum there, and one step of x itself
        # (the norm's own rounding may fall the other way)
        assert ((a.float() - b.float()).abs() <= (4 * 2.0 ** -8 + 2 * 2.0 ** -8) * size).all()
