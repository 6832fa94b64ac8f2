"""Shared prefixes and log probabilities where they are used: decode steps of the model over
groups of handles, the engine's requests behind prefixes with their tokens' log
probabilities, eager and replayed, and prompts scored without generating -- against the
fp32 oracle of the whole sequence (the bars of test_model_gpu.py)."""
import pytest
import torch

from conftest import announce
from test_chunk_model_gpu import _check_logits
from test_model_gpu import _pool, _tiny
from oracle import model as om

pytestmark = pytest.mark.gpu


def _forest(model, cfg, gpu, seed, blocks=220):
    """Handles behind two prefixes (one with a part of its own in common) and alone, in an
    order that mixes them: (pool, handles, their tokens)."""
    from qwen3_engine_from_scratch_amd.PagedKVcache import PagedKVCache, fork_caches

    g = torch.Generator().manual_seed(seed)

    def toks(n):
        return torch.randint(0, cfg.vocab_size, (n,), generator=g)

    pool = _pool(cfg, gpu, blocks=blocks, max_requests=40)
    bases = [toks(150), toks(33)]
    roots = [PagedKVCache(pool) for _ in bases]
    for r, b in zip(roots, bases):
        model.extend(b[None].to(gpu), r)
    from_root = [0, 1, 0, 0, 1, 0, 0, 0, 1, 0] * 2
    kids = fork_caches([roots[i] for i in from_root])
    tails = [toks(1 + 5 * (i % 7)) for i in range(len(kids))]
    seqs = [torch.cat((bases[i], t)) for i, t in zip(from_root, tails)]
    for _ in range(2):
        kids.append(PagedKVCache(pool))
        tails.append(toks(40))
        seqs.append(tails[-1])
    width = max(len(t) for t in tails)
    ids = torch.zeros(len(kids), width, dtype=torch.long)
    for i, t in enumerate(tails):
        ids[i, :len(t)] = t
    model.extend(ids.to(gpu), kids, [len(t) for t in tails])
    kids += fork_caches([kids[0]] * 2)  # behind a longer prefix than its own root's
    seqs += [seqs[0]] * 2
    return pool, kids, seqs


@pytest.mark.parametrize("fused", [False, True])
def test_decode_steps_over_groups(gpu, fused):
    from qwen3_engine_from_scratch_amd.PagedKVcache import (reserve_pages_bulk, set_seq_lens_bulk,
                                                            shared_prefix_groups)

    model, state, cfg = _tiny(seed=11)
    model = model.to(gpu)
    pool, kids, seqs = _forest(model, cfg, gpu, 21)
    announce(f"decode steps of {len(kids)} handles over shared prefixes, fused={fused}")
    order, *groups = shared_prefix_groups(kids)
    assert len(groups[1]) >= 2
    kids, seqs = [kids[i] for i in order], [seqs[i] for i in order]
    shared = tuple(torch.tensor(x, dtype=torch.int32, device=gpu) for x in groups)
    rows = torch.tensor([c.row_id for c in kids], dtype=torch.int32, device=gpu)
    g = torch.Generator().manual_seed(4)
    for step in range(2):
        more = torch.randint(0, cfg.vocab_size, (len(kids),), generator=g)
        reserve_pages_bulk(kids, [c.seq_len + 1 for c in kids])
        out = model.decode_logits(more.to(gpu), rows, pool, fused=fused, shared=shared)
        if not step:  # greedy tokens of the same step (it writes the same K/V again)
            toks = model.decode_greedy(more.to(gpu), rows, pool, shared=shared).cpu()
            best = out.max(dim=1).values.cpu()
            near = out.cpu()[torch.arange(len(kids)), toks]
            # the fused head sums in another order: near ties may fall otherwise
            assert (near >= best - 2 * torch.finfo(torch.bfloat16).eps * best.abs() - 0.05).all()
            again, logits = model.decode_greedy(more.to(gpu), rows, pool, shared=shared,
                                                with_logits=True)
            assert torch.equal(again.cpu(), toks) and torch.equal(
                logits, model.decode_logits(more.to(gpu), rows, pool, shared=shared))
        out = out.cpu()
        for c in kids:
            c.seq_len += 1
        set_seq_lens_bulk(kids)
        seqs = [torch.cat((s, t[None])) for s, t in zip(seqs, more)]
        for i, s in enumerate(seqs):
            _check_logits(out[i:i + 1], state, cfg, s, slice(-1, None), f"handle {i}.{step}")


@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("told", [None, 3])
def test_engine_over_shared_prefixes(gpu, use_graph, told):
    """Every token near the oracle's choice given the tokens before it (0.15 of that
    step's greatest logit, as test_model_gpu.py); its log probability within 0.3 of the
    oracle's (each logit within 0.15), and the listed tokens likewise."""
    from qwen3_engine_from_scratch_amd.engine import Engine, GenRequest

    model, state, cfg = _tiny(seed=3)
    model = model.to(gpu)
    g = torch.Generator().manual_seed(9)
    system = torch.randint(0, cfg.vocab_size, (83,), generator=g).tolist()
    more = system[:40] + torch.randint(0, cfg.vocab_size, (30,), generator=g).tolist()
    asks = [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist()
            for n in (5, 40, 1, 18, 9, 30, 2, 2, 13)]
    pool = _pool(cfg, gpu, blocks=160, max_requests=32)
    announce(f"engine with shared prefixes, graph={use_graph}, logprobs={told}")
    engine = Engine(model, pool, max_batch=6, use_graph=use_graph, share_prefixes=True)
    prefixes = [engine.cache_prefix(system), engine.cache_prefix(more)]
    reqs = [GenRequest(i, a, 3 + i % 5, prefix=[*prefixes, None][(0, 1, 0, 2, 0, 1, 0, 0, 1)[i]])
            for i, a in enumerate(asks)]
    for r in reqs[1::3]:
        r.logprobs = told
    if told:
        reqs[4].logprobs = 0
    engine.generate(reqs)
    for p in prefixes:
        p.free()
    assert not pool._extra_holders
    for r in reqs:
        prompt = (system if r.prefix is prefixes[0] else more if r.prefix is prefixes[1] else [])
        prompt = prompt + r.prompt
        assert len(r.output_ids) == r.max_new_tokens
        ref = om.qwen3_logits_ref(state, cfg, torch.tensor(prompt + r.output_ids)).double()
        logp = ref.log_softmax(-1)
        asked = len(r.output_ids) if r.logprobs is not None else 0
        assert len(r.output_logprobs) == len(r.output_top) == asked
        for k, tok in enumerate(r.output_ids):
            row = len(prompt) - 1 + k
            assert ref[row][tok] >= ref[row].max() - 0.15, (r.request_id, k)
            if asked:
                assert abs(r.output_logprobs[k] - logp[row][tok]) <= 0.3
                assert len(r.output_top[k]) == r.logprobs
                for i, lp in r.output_top[k]:
                    assert abs(lp - logp[row][i]) <= 0.3
                if r.logprobs:  # greedy: the first of the list, or near it
                    assert r.output_top[k][0][1] >= r.output_logprobs[k] \
                        >= r.output_top[k][0][1] - 0.3
    engine.close()


@pytest.mark.parametrize("share", [False, True])
def test_asking_changes_no_token(gpu, share):
    """The same requests, some of them asking for log probabilities or none: the same
    tokens, bit for bit, replayed or not."""
    from qwen3_engine_from_scratch_amd.engine import Engine, GenRequest

    model, state, cfg = _tiny(seed=13)
    model = model.to(gpu)
    g = torch.Generator().manual_seed(6)
    system = torch.randint(0, cfg.vocab_size, (70,), generator=g).tolist()
    asks = [torch.randint(0, cfg.vocab_size, (3 + i,), generator=g).tolist() for i in range(19)]
    announce(f"log probabilities asked for or not, shared prefixes {share}")
    told = []
    for ask in (None, 0, 5):
        pool = _pool(cfg, gpu, blocks=200, max_requests=64)
        engine = Engine(model, pool, max_batch=20, share_prefixes=share)
        prefix = engine.cache_prefix(system)
        reqs = [GenRequest(i, a, 4 + i, prefix=prefix if i % 4 else None)
                for i, a in enumerate(asks)]
        reqs[2].logprobs = reqs[14].logprobs = ask
        engine.generate(reqs)
        told.append([r.output_ids for r in reqs])
        prefix.free()
        engine.close()
    assert told[0] == told[1] == told[2]


def test_engines_of_both_modes_on_one_model(gpu):
    """Steps that are not replayed keep their engine's mode whatever engine was made last,
    and going to and fro takes no new workspaces."""
    from qwen3_engine_from_scratch_amd.engine import Engine, GenRequest

    model, state, cfg = _tiny(seed=15)
    model = model.to(gpu)
    g = torch.Generator().manual_seed(7)
    asks = [torch.randint(0, cfg.vocab_size, (40 + i,), generator=g).tolist() for i in range(5)]
    pool = _pool(cfg, gpu, blocks=120, max_requests=64)
    announce("a batch-invariant engine, a sharing and an eager one, in turn")
    exact = Engine(model, pool, max_batch=8, batch_invariant=True, max_prefill_batch=1)
    share = Engine(model, pool, max_batch=8, share_prefixes=True)
    eager = Engine(model, pool, max_batch=8, use_graph=False, share_prefixes=True)

    def run(engine, ask):
        reqs = [GenRequest(i, a, 6, logprobs=ask if i == 2 else None) for i, a in enumerate(asks)]
        engine.generate(reqs)
        return [r.output_ids for r in reqs]

    want, seen = None, None
    for _ in range(3):
        for ask in (None, 2):
            got = run(exact, ask)
            assert model._ws_mode is True or ask is None
            want = want or got
            assert got == want
            run(share, ask)
            run(eager, ask)
            assert model._ws_mode is False
        seen = seen or len(model._superseded)
        assert len(model._superseded) == seen
    for e in (exact, share, eager):
        e.close()


def test_sharing_changes_no_token_of_clear_choices(gpu):
    """The same requests with and without sharing: a token differs only where the oracle's
    two greatest logits are near each other (0.15, as above), and then the rest is not
    compared."""
    from qwen3_engine_from_scratch_amd.engine import Engine, GenRequest

    model, state, cfg = _tiny(seed=5)
    model = model.to(gpu)
    g = torch.Generator().manual_seed(2)
    system = torch.randint(0, cfg.vocab_size, (200,), generator=g).tolist()
    asks = [torch.randint(0, cfg.vocab_size, (3 + i,), generator=g).tolist() for i in range(40)]
    announce("40 requests behind one prefix, attended together or each by itself")
    told = []
    for share in (False, True):
        pool = _pool(cfg, gpu, blocks=400, max_requests=150)
        engine = Engine(model, pool, max_batch=48, share_prefixes=share)
        prefix = engine.cache_prefix(system)
        reqs = [GenRequest(i, a, 5, prefix=prefix) for i, a in enumerate(asks)]
        engine.generate(reqs)
        told.append([r.output_ids for r in reqs])
        prefix.free()
        engine.close()
    for a, x, y in zip(asks, *told):
        if x != y:
            k = next(i for i in range(5) if x[i] != y[i])
            ref = om.qwen3_logits_ref(state, cfg, torch.tensor(system + a + x))
            top = ref[len(system) + len(a) - 1 + k].topk(2).values
            assert top[0] - top[1] <= 0.15


def test_score(gpu):
    """Log probabilities, entropies and likely tokens of prompts against the oracle's
    logits (each within 0.15: 0.3 of a log probability; of an entropy sum |dp| log p <= 0.3 *
    (1 + the largest |log p|))."""
    from qwen3_engine_from_scratch_amd.engine import Engine

    model, state, cfg = _tiny(seed=6)
    model = model.to(gpu)
    g = torch.Generator().manual_seed(8)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist()
               for n in (1, 7, 130, 2, 64, 1, 30)]
    pool = _pool(cfg, gpu)
    engine = Engine(model, pool, max_batch=2, use_graph=False)
    announce("prompts scored, in batches of up to 100 tokens and all at once")
    free = pool.free_count, len(pool._free_rows)
    runs = [engine.score(prompts, top_n=4, entropy=True, max_tokens=n) for n in (100, 8192)]
    assert (pool.free_count, len(pool._free_rows)) == free
    for got in runs:
        assert len(got) == len(prompts)
        for p, s in zip(prompts, got):
            n = len(p) - 1
            assert s.logprobs.shape == (n,) and s.entropy.shape == (n,)
            assert s.top_ids.shape == (n, 4) and s.top_logprobs.shape == (n, 4)
            logp = om.qwen3_logits_ref(state, cfg, torch.tensor(p)).double().log_softmax(-1)[:n]
            want = logp.gather(1, torch.tensor(p[1:], dtype=torch.long)[:, None])[:, 0]
            assert (s.logprobs - want).abs().le(0.3).all()
            assert (s.top_logprobs - logp.gather(1, s.top_ids)).abs().le(0.3).all()
            assert (s.top_logprobs[:, :1] >= s.top_logprobs).all()
            ent = -(logp.exp() * logp).sum(1)
            assert ((s.entropy - ent).abs() <= 0.3 * (1 + logp.abs().amax(1))).all()
    only = engine.score(prompts[2:3])[0]
    assert only.entropy is None and only.top_ids is None
    # the same rows in another batch: the library products round otherwise, as above
    assert (only.logprobs - runs[0][2].logprobs).abs().le(0.3).all()
    assert engine.score([]) == []
    for bad in ([[]], [[1] * 1025]):
        with pytest.raises(ValueError):
            engine.score(bad)
    engine.close()
