"""Decode attention over shared prefixes against its definition in 64 bits (each sequence
by itself, oracle/chunk.py): groups, lengths at tile and page borders, sequences shorter
than their prefix, empty ones, bad pages, strides, streams and graphs."""
import pytest
import torch

from conftest import announce
from oracle.chunk import paged_chunk_ref
from test_chunk_precision_gpu import bound

pytestmark = pytest.mark.gpu

SCALE = 128 ** -0.5


def make_shared(groups, hq, hkv, bs, dev, *, seed=0, std=2.0, layers=2, slack_rows=3, extra_pages=1):
    """groups: (tokens of the prefix, tokens of each sequence behind it).  The prefix's
    whole pages are shared, a partly filled one is each sequence's own (as forks have it).
    Every slot that is no token's holds NaN.  seq_lens are lengths before the step."""
    g = torch.Generator(device=dev).manual_seed(seed)
    gc = torch.Generator().manual_seed(seed)
    B, D = sum(len(o) for _, o in groups), 128
    rows = B + slack_rows
    width = max(max(-(-(p + n) // bs) for p, own in groups for n in own), 1) + extra_pages
    blocks = sum(p // bs + sum(-(-(p + n) // bs) - p // bs for n in own) for p, own in groups) + 3
    perm = torch.randperm(blocks, generator=gc).tolist()
    pools = [torch.full((blocks, layers, hkv, bs, D), float("nan"), dtype=torch.bfloat16, device=dev)
             for _ in range(2)]
    table = torch.full((rows, width), -1, dtype=torch.int32)
    row_ids = torch.randperm(rows, generator=gc)[:B].to(torch.int32)
    seq_lens = torch.randint(0, 50, (rows,), generator=gc).to(torch.int32)

    def fill(ids, tokens):
        for x in pools:
            new = torch.empty(len(ids), hkv, bs, D, dtype=torch.bfloat16, device=dev).normal_(generator=g)
            if len(ids) and tokens < len(ids) * bs:
                new[-1, :, tokens - (len(ids) - 1) * bs:] = float("nan")
            x[torch.tensor(ids, dtype=torch.long, device=dev), layers - 1] = new

    b, cu, shared = 0, [0], []
    for p, own in groups:
        pre = [perm.pop() for _ in range(p // bs)]
        fill(pre, len(pre) * bs)
        for n in own:
            mine = [perm.pop() for _ in range(-(-(p + n) // bs) - len(pre))]
            fill(mine, p + n - len(pre) * bs)
            r = int(row_ids[b])
            table[r, :len(pre) + len(mine)] = torch.tensor(pre + mine, dtype=torch.int32)
            seq_lens[r] = p + n - 1
            b += 1
        cu.append(b)
        shared.append(p // bs * bs)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    q = torch.empty(B, hq, D, dtype=torch.bfloat16, device=dev).normal_(0.0, std, generator=g)
    return dict(q=q, k=pools[0][:, layers - 1], v=pools[1][:, layers - 1], table=table,
                seq_lens=seq_lens, row_ids=row_ids, groups=i32(cu), shared=i32(shared), bs=bs,
                cu=torch.arange(B + 1))


def run(t, dev, **kw):
    from qwen3_engine_from_scratch_amd.kernels.paged_attention import paged_attention_decode_shared_hip

    rows = t["row_ids"]
    return paged_attention_decode_shared_hip(
        t["q"], t["k"], t["v"], t["table"].to(dev), t["seq_lens"].to(dev),
        None if rows is None else rows.to(dev), t["groups"].to(dev), t["shared"].to(dev), t["bs"], **kw)


def check(out, t, what, scale=SCALE):
    """bound() counts the errors of weights in 16 bits over n keys; joins add a weight, a
    product and a sum for each part, inside the 2 n + 4 steps that it allows."""
    ref, spread = paged_chunk_ref(t["q"], t["k"], t["v"], t["table"], t["seq_lens"], t["row_ids"],
                                  t["cu"], t["bs"], scale)
    assert torch.isfinite(out).all(), f"{what}: non-finite output"
    known = t["row_ids"].clamp(0, t["table"].shape[0] - 1)  # (others hold no keys)
    over = (out.double() - ref).abs() - bound(dict(t, row_ids=known), ref, spread)
    print(f"[err] {what}: max-abs {(out.double() - ref).abs().max().item():.3e}, worst excess "
          f"{over.max().item():.3e}", flush=True)
    assert over.max() <= 0, what


SHAPES = [
    # groups, query heads, KV heads, block size
    ([(64, [1])], 16, 8, 16),                                  # a group of one
    ([(64, [5, 7])], 16, 8, 16),                               # four rows: streamed
    ([(64, [1] * 8)], 16, 8, 16),                              # sixteen rows
    ([(64, [1] * 9)], 16, 8, 16),                              # eighteen: staged
    ([(896, [3, 40, 17, 1])], 16, 8, 16),
    ([(16, [1] * 40)], 8, 8, 16),                              # one tile of sixteen
    ([(15, [3, 4])], 16, 8, 16),                               # nothing to share
    ([(100, list(range(1, 20)))], 32, 8, 16),                  # a partly filled page
    ([(4096, [10, 600, 333] * 5)], 32, 8, 16),
    ([(1000, [5, 9, 2, 700, 31, 64, 65])], 40, 8, 16),         # five heads a group
    ([(2000, [1 + 37 * i % 90 for i in range(70)])], 32, 8, 16),  # two row tiles
    ([(500, [1 + i for i in range(110)])], 40, 8, 16),         # a sequence across row tiles
    ([(777, [4] * 20)], 16, 1, 16),                            # sixteen heads
    ([(320, [9, 200, 1])], 6, 2, 32),
    ([(480, [50, 1, 2] * 8)], 16, 8, 48),
    ([(640, [64, 63, 65] * 4)], 16, 2, 64),
    ([(500, [7] * 5), (0, [900]), (1200, [3] * 30), (48, [11, 2]), (0, [1]), (64, [400])], 16, 8, 16),
    ([(3000, [20] * 12), (5000, [100] * 3), (100, [1] * 40), (12000, [900] * 5)], 16, 8, 32),
    ([(2000, [50 + 9 * i for i in range(256)])], 16, 8, 16),
    ([(0, [i + 1 for i in range(30)])], 16, 8, 16),            # no prefix
]


@pytest.mark.parametrize("groups,hq,hkv,bs", SHAPES)
def test_against_the_definition(gpu, groups, hq, hkv, bs):
    what = f"{[(p, len(o)) for p, o in groups]} heads {hq}/{hkv} blocks of {bs}"
    announce("shared " + what)
    t = make_shared(groups, hq, hkv, bs, gpu, seed=hq + len(groups))
    out = run(t, gpu)
    torch.cuda.synchronize()
    check(out, t, what)
    assert torch.equal(run(t, gpu), out), "the same call gave other bits"


def test_probabilities_keep_sixteen_bits(gpu):
    """Few keys and small scores: a single bf16 rounding of P would show."""
    for n, p, hq in ((6, 16, 32), (20, 16, 32), (80, 32, 16)):
        announce(f"shared precision: {n} sequences behind {p}")
        t = make_shared([(p, [1, 2, 5] * (n // 3) + [1] * (n % 3))], hq, 8, 16, gpu, seed=n, std=0.25)
        check(run(t, gpu), t, f"{n} behind {p}")


def test_long_prefixes(gpu):
    for groups, hq, hkv in (([(100000, [30, 400, 1, 77] * 8)], 32, 8), ([(70001, [3, 90])], 16, 8),
                            ([(30000, [10] * 33), (45000, [700] * 2)], 8, 2)):
        announce(f"shared long {[(p, len(o)) for p, o in groups]}")
        t = make_shared(groups, hq, hkv, 16, gpu, seed=5)
        out = run(t, gpu)
        torch.cuda.synchronize()
        check(out, t, "long prefixes")


@pytest.mark.parametrize("B,per", [(1024, 1024), (1000, 3), (700, 1), (520, 130), (1023, 2)])
def test_many_sequences(gpu, B, per):
    announce(f"shared: {B} sequences in groups of {per}")
    g = torch.Generator().manual_seed(B)
    own = torch.randint(1, 60, (B,), generator=g).tolist()
    groups = [(16 * (i % 7), own[i:i + per]) for i in range(0, B, per)]
    t = make_shared(groups, 16, 8, 16, gpu, seed=B)
    out = run(t, gpu)
    torch.cuda.synchronize()
    check(out, t, f"{B} sequences")


@pytest.mark.parametrize("n", [5, 12, 70])
def test_lengths_inside_the_prefix(gpu, n):
    """Sequences that end inside the shared positions (the first one too), or hold nothing."""
    announce(f"shared: {n} sequences, some shorter than their prefix")
    t = make_shared([(300, [20] * n), (200, [1, 2])], 32, 8, 16, gpu, seed=n)
    rows = t["row_ids"].long()
    for i, length in ((1, 287), (2, 0), (3, 16), (4, 17), (n, 5)):
        t["seq_lens"][rows[i]] = length - 1
    check(run(t, gpu), t, "shorter than the prefix")
    t["seq_lens"][rows[0]] = 99  # the prefix counts as far as the first one goes
    check(run(t, gpu), t, "the first one shorter")
    t["seq_lens"][rows[0]] = -1
    out = run(t, gpu)
    check(out, t, "the first one empty")
    assert not out[0].any() and not out[2].any()
    t["seq_lens"][rows] = -7
    assert not run(t, gpu).any()


@pytest.mark.parametrize("n", [4, 30])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_values_behind_a_sequences_end(gpu, n, bad):
    """What the shared pages hold behind the end of a sequence that is shorter than its
    group's prefix does not reach it: the same bits whatever stands there."""
    announce(f"shared: {n} sequences, {bad} behind the end of some")
    t = make_shared([(320, [20] * n)], 16, 4, 16, gpu, seed=n)
    rows = t["row_ids"].long()
    short = [1, 2, n - 1]
    for i, length in zip(short, (288, 7, 290)):
        t["seq_lens"][rows[i]] = length - 1
    clean = run(t, gpu)
    check(clean, t, "clean")
    page = int(t["table"][rows[0], 18])  # tokens 288 .. 303
    for x in (t["k"], t["v"]):
        x[page, :, 2:] = bad
    out = run(t, gpu)
    assert torch.equal(out[short], clean[short])


def test_claims_of_odd_lengths(gpu):
    """shared_lens inside a page or a tile, beyond the first sequence, none, negative."""
    announce("shared: claims of odd lengths")
    t = make_shared([(640, [30] * 9), (640, [5, 6])], 32, 8, 64, gpu, seed=2)
    for claim in (639, 600, 97, 17, 16, 15, 1, 0, -5, -2 ** 31):
        t["shared"] = torch.tensor([claim, claim], dtype=torch.int32)
        check(run(t, gpu), t, f"claim {claim}")
    t = make_shared([(640, [0] * 9), (640, [0, 0])], 32, 8, 64, gpu, seed=2)  # nothing of their own
    t["shared"] = torch.tensor([2 ** 31 - 1, 2 ** 31 - 1], dtype=torch.int32)
    check(run(t, gpu), t, "all shared, a claim beyond")


def test_groups_that_are_no_ranges(gpu):
    """Entries before, between (empty groups) and behind the groups attend alone; bounds
    outside the batch count as no group."""
    announce("shared: odd groups")
    t = make_shared([(0, [9, 70]), (320, [3] * 12), (0, [5, 1, 300])], 16, 8, 16, gpu, seed=3)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    for cu, shared in (([2, 14], [320]), ([2, 2, 14, 14], [5, 320, 99]), ([2, 8, 14], [320, 320]),
                       ([0, 2, 14, 17], [0, 320, 0]), ([2, 14, 18], [320, 64]), ([14, 2], [320]),
                       ([-1, 14], [320]), ([2, 2 ** 31 - 1], [320]), ([0], [])):
        t["groups"], t["shared"] = i32(cu), i32(shared)
        check(run(t, gpu), t, f"groups {cu}")


def test_rows_and_pages_outside(gpu):
    announce("shared: rows outside the table, pages outside the pool")
    t = make_shared([(400, [20] * 12), (300, [4, 5])], 16, 8, 16, gpu, seed=4)
    rows = t["row_ids"].long()
    blocks = t["k"].shape[0]
    for page, bad in ((3, -1), (9, blocks), (20, 2 ** 31 - 1), (21, -2 ** 31)):
        t["table"][rows[:12], page] = bad
    t["table"][rows[12], 2] = blocks + 5
    t["table"][rows[13], 2] = blocks + 5
    t["table"][rows[3], 25] = blocks
    check(run(t, gpu), t, "bad pages")
    t["row_ids"] = t["row_ids"].clone()
    t["row_ids"][5], t["row_ids"][13] = 10 ** 6, -1
    out = run(t, gpu)
    check(out, t, "bad rows")
    assert not out[5].any() and not out[13].any()
    t["row_ids"][0] = -1  # a group whose first sequence has no row attends alone
    check(run(t, gpu), t, "the first row bad")
    t = make_shared([(400, [20] * 12)], 16, 8, 16, gpu, seed=4)
    t["table"] = t["table"][:, :22].contiguous()  # positions behind the table's rows
    t["shared"] = torch.tensor([384], dtype=torch.int32)
    check(run(t, gpu), t, "short rows")


def test_no_row_ids_and_bias(gpu):
    announce("shared: rows 0 .. B - 1, another bias, scale")
    t = make_shared([(96, [5] * 11)], 16, 8, 16, gpu, seed=6, slack_rows=0)
    order = torch.argsort(t["row_ids"].long())
    t["table"] = t["table"][t["row_ids"].long()].contiguous()
    t["seq_lens"] = t["seq_lens"][t["row_ids"].long()].contiguous()
    t["row_ids"] = torch.arange(11, dtype=torch.int32)
    assert len(order) == 11
    ref = run(t, gpu)
    check(ref, t, "row ids")
    own = dict(t, row_ids=None)
    assert torch.equal(run(own, gpu), ref)
    longer = dict(t, seq_lens=t["seq_lens"] + 1)
    assert torch.equal(run(longer, gpu, seq_len_bias=0), ref)
    check(run(t, gpu, scale=0.02), t, "scale", scale=0.02)


@pytest.mark.parametrize("n", [3, 20])
def test_strided_views(gpu, n):
    announce(f"shared: strided views, {n} sequences")
    t = make_shared([(200, [7] * n)], 16, 8, 16, gpu, seed=7, layers=3)
    wide = torch.zeros(n, 40 * 128, dtype=torch.bfloat16, device=gpu)
    wide[:, 128:128 + 16 * 128] = t["q"].reshape(n, -1)
    t["q"] = wide[:, 128:128 + 16 * 128].view(n, 16, 128)
    hold = torch.full((n, 2, 16, 128), 3.0, dtype=torch.bfloat16, device=gpu)
    assert run(t, gpu, out=hold[:, 1]).data_ptr() == hold[:, 1].data_ptr()
    check(hold[:, 1], t, "strided")
    assert (hold[:, 0] == 3.0).all()
    t["q"] = t["q"].transpose(0, 1).contiguous().transpose(0, 1)
    check(run(t, gpu), t, "head-major q")


def test_large_scores(gpu):
    announce("shared: large scores")
    t = make_shared([(300, [9] * 20), (150, [40, 2])], 16, 8, 16, gpu, seed=9, std=30.0)
    check(run(t, gpu), t, "large scores")


def test_agrees_with_decode(gpu):
    """The same attention as paged_attention_decode_hip, both within the bound; alone it
    is the same loop."""
    from qwen3_engine_from_scratch_amd.kernels.paged_attention import paged_attention_decode_hip

    announce("shared against decode")
    t = make_shared([(512, [1, 30, 200] * 8), (0, [77])], 32, 8, 16, gpu, seed=10)
    dec = paged_attention_decode_hip(t["q"], t["k"], t["v"], t["table"].to(gpu),
                                     t["seq_lens"].to(gpu), t["row_ids"].to(gpu), 16)
    check(dec, t, "decode")
    check(run(t, gpu), t, "shared")


def test_nothing_to_do(gpu):
    t = make_shared([(32, [1, 2])], 16, 8, 16, gpu)
    t.update(q=t["q"][:0], row_ids=t["row_ids"][:0], groups=t["groups"][:1], shared=t["shared"][:0])
    assert run(t, gpu).shape == (0, 16, 128)


def test_capture_and_replay_with_other_groups(gpu):
    announce("shared: captured, replayed with other lengths and groups")
    from qwen3_engine_from_scratch_amd.kernels.paged_attention import paged_attention_decode_shared_hip

    t = make_shared([(400, [20] * 12), (300, [4, 50, 300])], 16, 8, 16, gpu, seed=11)
    dev = {k: t[k].to(gpu) for k in ("table", "seq_lens", "row_ids", "groups", "shared")}
    q, out = t["q"].clone(), torch.empty_like(t["q"])

    def call():
        paged_attention_decode_shared_hip(q, t["k"], t["v"], dev["table"], dev["seq_lens"],
                                          dev["row_ids"], dev["groups"], dev["shared"], 16, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    plans = [([0, 12, 15], [400, 300]), ([0, 3, 12], [400, 64]), ([0, 12, 12], [16, 0]), ([0, 0, 0], [0, 0])]
    for i, (cu, shared) in enumerate(plans):
        t["groups"], t["shared"] = i32(cu), i32(shared)
        t["seq_lens"][t["row_ids"].long()[i]] -= 11 * i
        for k in ("groups", "shared", "seq_lens"):
            dev[k].copy_(t[k])
        q.normal_(0.0, 2.0)
        t["q"] = q
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        check(out, t, f"replay {i}")
        got = out.clone()
        torch.empty(1 << 24, device=gpu).normal_()  # eager work between the replays
        call()
        torch.cuda.synchronize()
        assert torch.equal(got, out), f"replay {i} differs from the eager call"


def test_calls_on_two_streams(gpu):
    announce("shared: two streams at once")
    cases = [make_shared([(3000, [40] * 30)], 16, 8, 16, gpu, seed=12),
             make_shared([(500, [4, 5, 1000])], 16, 8, 16, gpu, seed=13)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[], []]
    for _ in range(6):
        for i, (t, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                outs[i].append(run(t, gpu))
    torch.cuda.synchronize()
    for i, t in enumerate(cases):
        check(outs[i][0], t, f"stream {i}")
        for o in outs[i][1:]:
            assert torch.equal(o, outs[i][0]), "the same call gave other bits"


def test_a_workspace_of_the_callers(gpu):
    from qwen3_engine_from_scratch_amd.kernels.paged_attention import paged_decode_shared_workspace_bytes

    announce("shared: workspace filled with garbage")
    t = make_shared([(300, [40] * 30), (64, [1, 2])], 16, 8, 16, gpu, seed=14)
    ws = torch.full((paged_decode_shared_workspace_bytes(32, 16, 8, 128),), 255, dtype=torch.uint8, device=gpu)
    check(run(t, gpu, workspace=ws), t, "garbage workspace")


def test_far_blocks(gpu):
    """Pages beyond 2^31 elements of the pool."""
    blocks_all, layers = 5000, 28
    t = make_shared([(320, [9] * 20), (160, [3, 50])], 32, 8, 16, gpu, seed=15)
    blocks = t["k"].shape[0]
    big = [torch.empty(blocks_all, layers, 8, 16, 128, dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    assert big[0].numel() > 1 << 31
    announce("shared: the last blocks of a large pool")
    for x, name in zip(big, ("k", "v")):
        x[blocks_all - blocks:, layers - 1] = t[name]
    moved = dict(t, k=big[0][:, layers - 1], v=big[1][:, layers - 1],
                 table=torch.where(t["table"] >= 0, t["table"] + (blocks_all - blocks), -1))
    check(run(moved, gpu), t, "far blocks")
