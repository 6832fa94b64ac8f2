"""Attention of a chunk of new tokens over the paged cache against its definition in
64 bits (oracle/chunk.py): shapes, empty rows, bad pages, lengths at tile and page
borders, strides, streams and graphs."""
import pytest
import torch

from conftest import announce
from oracle.chunk import paged_chunk_ref

pytestmark = pytest.mark.gpu


def make_case(chunks, ctxs, hq, hkv, bs, dev, *, seed=0, slack_rows=2, extra_pages=0, layers=2,
              std=2.0, tail=0):
    """A pool of `layers` layers whose every slot that is no token's holds NaN; each
    sequence's pages lie scattered.  tail: rows of q behind the last sequence."""
    g = torch.Generator(device=dev).manual_seed(seed)
    gc = torch.Generator().manual_seed(seed)
    B, D = len(chunks), 128
    lens = [n + max(c, 0) for n, c in zip(chunks, ctxs)]
    pages = [-(-L // bs) for L in lens]
    blocks = sum(pages) + 3
    perm = torch.randperm(blocks, generator=gc).to(torch.int32)
    rows = B + slack_rows
    width = max(max(pages), 1) + extra_pages
    table = torch.full((rows, width), -1, dtype=torch.int32)
    row_ids = torch.randperm(rows, generator=gc)[:B].to(torch.int32)
    seq_lens = torch.randint(0, 50, (rows,), generator=gc).to(torch.int32)
    pools = [torch.full((blocks, layers, hkv, bs, D), float("nan"), dtype=torch.bfloat16, device=dev)
             for _ in range(2)]
    off = 0
    for b, (p, L) in enumerate(zip(pages, lens)):
        r = int(row_ids[b])
        table[r, :p] = perm[off:off + p]
        seq_lens[r] = ctxs[b]
        idx = perm[off:off + p].long().to(dev)
        for x in pools:
            new = torch.empty(p, hkv, bs, D, dtype=torch.bfloat16, device=dev)
            new.normal_(0.0, 1.0, generator=g)
            used = L - (p - 1) * bs
            if p and used < bs:
                new[-1, :, used:] = float("nan")
            x[idx, layers - 1] = new
        off += p
    cu = torch.zeros(B + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(chunks, dtype=torch.int32).cumsum(0)
    T = int(cu[-1]) + tail
    q = torch.empty(T, hq, D, dtype=torch.bfloat16, device=dev).normal_(0.0, std, generator=g)
    return dict(q=q, k=pools[0][:, layers - 1], v=pools[1][:, layers - 1], table=table,
                seq_lens=seq_lens, row_ids=row_ids, cu=cu, bs=bs, most=max(chunks, default=0))


def run(t, dev, **kw):
    from qwen3_engine_from_scratch_amd.kernels.paged_attention import paged_attention_chunk_hip

    kw.setdefault("max_chunk", t["most"])
    return paged_attention_chunk_hip(t["q"], t["k"], t["v"], t["table"].to(dev),
                                     t["seq_lens"].to(dev), t["row_ids"].to(dev),
                                     t["cu"].to(dev), t["bs"], **kw)


def check(out, t, what, scale=128 ** -0.5):
    """|out - o| <= 2^-8 (spread + |o|): P is rounded to bf16 before it meets V (half a
    step, 2^-8 of each term: 2^-8 sum p |v|), and the output once more (2^-8 |o|, of the
    value with the first error in it: 2^-16 spread).  fp32 scores and sums: a score of
    128 products is off by at most 128 2^-24 |q| |k| scale, below 2^-24 128 * 40 = 3e-4
    at these |q k| (and so P), the exponential by 2^-22, the sums over n keys in parts of 64
    by a few 2^-24: together below 2^-10 spread."""
    ref, spread = paged_chunk_ref(t["q"], t["k"], t["v"], t["table"], t["seq_lens"], t["row_ids"],
                                  t["cu"], t["bs"], scale)
    n = int(t["cu"][-1])
    o, r, w = out[:n].double(), ref[:n], spread[:n]
    assert torch.isfinite(o).all(), f"{what}: non-finite output"
    over = (o - r).abs() - (2.0 ** -8 * (w * (1 + 2.0 ** -8) + r.abs()) + 2.0 ** -10 * w + 1e-30)
    d = (o - r).abs().max().item() if n else 0.0
    print(f"[err] {what}: max-abs {d:.3e}, worst excess {over.max().item() if n else 0.0:.3e}",
          flush=True)
    assert n == 0 or over.max() <= 0, what


SHAPES = [
    # chunks, cached tokens, query heads, KV heads, block size
    ([5], [0], 16, 8, 16),
    ([1], [0], 8, 8, 16),
    ([1], [63], 32, 8, 16),
    ([5], [900], 16, 8, 16),
    ([4, 4, 4], [100, 17, 1000], 32, 8, 16),
    ([1, 1, 1, 1], [15, 16, 17, 64], 16, 8, 16),
    ([3, 0, 2], [40, 9, 0], 16, 8, 32),
    ([16, 9, 1], [333, 48, 2], 16, 8, 16),          # 32 packed rows a KV head
    ([17, 2], [200, 0], 16, 8, 16),                  # 34
    ([64], [0], 16, 8, 16),
    ([65, 1, 127], [63, 64, 65], 16, 8, 16),
    ([100, 300, 7], [1, 500, 2000], 32, 8, 16),
    ([33, 129, 2], [7, 0, 130], 8, 8, 16),           # one head a group
    ([40, 70], [90, 3], 6, 2, 16),                   # three
    ([50, 21], [33, 256], 40, 8, 16),                # five
    ([31, 90], [400, 15], 16, 2, 64),                # eight
    ([11, 20], [70, 0], 16, 1, 48),                  # sixteen, blocks of 48
    ([500], [3000], 32, 8, 32),
    ([1, 257, 1, 1, 30], [700, 100, 33, 2500, 0], 16, 8, 16),  # decoding beside prefilling
]


@pytest.mark.parametrize("chunks,ctxs,hq,hkv,bs", SHAPES)
def test_chunk_against_its_definition(gpu, chunks, ctxs, hq, hkv, bs):
    announce(f"chunk {chunks} behind {ctxs} heads {hq}/{hkv} blocks of {bs}")
    t = make_case(chunks, ctxs, hq, hkv, bs, gpu, seed=sum(chunks) + hq)
    out = run(t, gpu)
    torch.cuda.synchronize()
    check(out, t, f"{chunks} behind {ctxs}")


def test_long_contexts(gpu):
    for chunks, ctxs, hq, hkv in (([40], [100000], 32, 8), ([3, 2], [70000, 33333], 16, 8),
                                  ([260], [30011], 16, 8)):
        announce(f"chunk {chunks} behind {ctxs}")
        t = make_case(chunks, ctxs, hq, hkv, 16, gpu, seed=5)
        out = run(t, gpu)
        torch.cuda.synchronize()
        check(out, t, f"{chunks} behind {ctxs}")


def test_many_sequences(gpu):
    g = torch.Generator().manual_seed(3)
    for B, hi, far in ((300, 3, 90), (70, 40, 300), (2100, 1, 40)):
        chunks = torch.randint(0, hi + 1, (B,), generator=g).tolist()
        ctxs = torch.randint(0, far, (B,), generator=g).tolist()
        announce(f"{B} sequences of up to {hi} new tokens")
        t = make_case(chunks, ctxs, 16, 8, 16, gpu, seed=B)
        out = run(t, gpu)
        torch.cuda.synchronize()
        check(out, t, f"{B} sequences")


@pytest.mark.parametrize("chunks,ctxs", [([3, 2], [20, 90]), ([70, 130], [20, 90])])
def test_rows_of_no_sequence_are_left_and_rows_without_keys_are_zero(gpu, chunks, ctxs):
    announce(f"chunk {chunks}: rows behind the last sequence, rows without keys")
    t = make_case(chunks + [4, 5], ctxs + [-4, 30], 16, 8, 16, gpu, seed=1, tail=9)
    t["row_ids"][-1] = 10 ** 6  # no row of the table
    out = torch.full_like(t["q"], 7.0)
    assert run(t, gpu, out=out) is out
    torch.cuda.synchronize()
    n = int(t["cu"][-1])
    assert (out[n:] == 7.0).all()
    assert not out[n - 5:n].any(), "a sequence without a row"
    assert not out[n - 9:n - 5].any(), "positions -4 .. -1"
    check(out, t, "rows without keys")


@pytest.mark.parametrize("chunks,ctxs", [([3, 5], [500, 90]), ([70, 130], [400, 90])])
def test_pages_outside_the_pool_are_not_attended(gpu, chunks, ctxs):
    announce(f"chunk {chunks}: bad page ids")
    t = make_case(chunks, ctxs, 16, 8, 16, gpu, seed=2)
    blocks = t["k"].shape[0]
    r0, r1 = int(t["row_ids"][0]), int(t["row_ids"][1])
    t["table"][r0, 3] = -1
    t["table"][r0, 7] = blocks
    t["table"][r1, 0] = 2 ** 31 - 1
    t["table"][r1, 4] = -(2 ** 31)
    out = run(t, gpu)
    torch.cuda.synchronize()
    check(out, t, "bad page ids")


@pytest.mark.parametrize("n", [2, 90])
def test_a_table_row_that_ends_before_the_sequence(gpu, n):
    announce(f"chunk of {n}: positions behind the table row")
    t = make_case([n, n], [200, 30], 16, 8, 16, gpu, seed=4)
    t["table"] = t["table"][:, :9].contiguous()  # 144 positions
    out = run(t, gpu)
    torch.cuda.synchronize()
    check(out, t, "short table row")


@pytest.mark.parametrize("chunks,ctxs", [([4, 1], [90, 3]), ([90, 41], [65, 0])])
def test_strided_views(gpu, chunks, ctxs):
    announce(f"chunk {chunks}: slices of a fused projection, strided output")
    t = make_case(chunks, ctxs, 16, 8, 16, gpu, seed=6, layers=3)
    T = t["q"].shape[0]
    wide = torch.randn(T, 40 * 128, device=gpu).to(torch.bfloat16)
    wide[:, 128:128 + 16 * 128] = t["q"].reshape(T, -1)
    t["q"] = wide[:, 128:128 + 16 * 128].view(T, 16, 128)
    hold = torch.full((T, 2, 16, 128), 3.0, dtype=torch.bfloat16, device=gpu)
    out = run(t, gpu, out=hold[:, 1])
    torch.cuda.synchronize()
    check(out, t, "strided")
    assert (hold[:, 0] == 3.0).all()
    # heads of q in another order of the axes
    t["q"] = t["q"].transpose(0, 1).contiguous().transpose(0, 1)
    check(run(t, gpu), t, "head-major q")


def test_scale_and_bounds(gpu):
    announce("chunk: another scale, a loose max_chunk, max_chunk from cu_seqlens")
    for chunks, ctxs in (([3, 1], [50, 200]), ([80, 33], [50, 200])):
        t = make_case(chunks, ctxs, 16, 8, 16, gpu, seed=8)
        check(run(t, gpu, scale=0.02), t, "scale 0.02", scale=0.02)
        check(run(t, gpu, max_chunk=4000), t, "loose bound")
        check(run(t, gpu, max_chunk=None), t, "bound read back")


def test_large_scores(gpu):
    """Scores of several hundred units: the running maximum must keep up."""
    announce("chunk: large scores")
    for chunks, ctxs in (([3, 1], [50, 700]), ([80, 33], [50, 700])):
        t = make_case(chunks, ctxs, 16, 8, 16, gpu, seed=9, std=30.0)
        out = run(t, gpu)
        ref, spread = paged_chunk_ref(t["q"], t["k"], t["v"], t["table"], t["seq_lens"],
                                      t["row_ids"], t["cu"], 16, 128 ** -0.5)
        # |q k| scale up to 30 * 5 * 11: a score is off by 128 2^-24 * 1900 = 1.5e-2 at the
        # very most, and so are the weights
        assert ((out.double() - ref).abs() <= (2.0 ** -8 + 2 * 1.5e-2) * (spread + ref.abs())).all()


def test_single_tokens_agree_with_decode(gpu):
    from qwen3_engine_from_scratch_amd.kernels.paged_attention import paged_attention_decode_hip

    announce("chunks of one token against paged decode")
    t = make_case([1] * 5, [0, 15, 16, 700, 3000], 32, 8, 16, gpu, seed=10)
    out = run(t, gpu)
    dec = paged_attention_decode_hip(t["q"], t["k"], t["v"], t["table"].to(gpu),
                                     t["seq_lens"].to(gpu), t["row_ids"].to(gpu), 16)
    _, spread = paged_chunk_ref(t["q"], t["k"], t["v"], t["table"], t["seq_lens"], t["row_ids"],
                                t["cu"], 16, 128 ** -0.5)
    # each is within the bound of check() of the same values
    bound = 2 * (2.0 ** -8 * (spread * (1 + 2.0 ** -8) + out.double().abs() + 2.0 ** -8 * spread)
                 + 2.0 ** -10 * spread)
    assert ((out.double() - dec.double()).abs() <= bound).all()


@pytest.mark.parametrize("chunks,ctxs", [([4, 1, 3], [900, 40, 0]), ([200, 1, 64], [900, 40, 0])])
def test_capture_and_replay_with_other_lengths(gpu, chunks, ctxs):
    announce(f"chunk {chunks}: captured, replayed with other lengths and tables")
    t = make_case(chunks, ctxs, 16, 8, 16, gpu, seed=11, extra_pages=2)
    dev = {k: t[k].to(gpu) for k in ("table", "seq_lens", "row_ids", "cu")}
    from qwen3_engine_from_scratch_amd.kernels.paged_attention import paged_attention_chunk_hip

    q, out = t["q"].clone(), torch.empty_like(t["q"])

    def call():
        paged_attention_chunk_hip(q, t["k"], t["v"], dev["table"], dev["seq_lens"],
                                  dev["row_ids"], dev["cu"], 16, max_chunk=t["most"], out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(4):
        r = int(t["row_ids"][i % 3])
        t["seq_lens"][r] = max(0, int(t["seq_lens"][r]) - 13 * i)
        dev["seq_lens"].copy_(t["seq_lens"])
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
    announce("chunk: two streams at once")
    cases = [make_case([200, 3], [3000, 100], 16, 8, 16, gpu, seed=12),
             make_case([3, 2], [5000, 3000], 16, 8, 16, gpu, seed=13)]
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


def test_nothing_to_do(gpu):
    announce("chunk: no tokens, no sequences")
    t = make_case([0, 0], [5, 0], 16, 8, 16, gpu)
    assert run(t, gpu).shape == (0, 16, 128)
    t = make_case([3], [5], 16, 8, 16, gpu)
    t.update(cu=torch.zeros(1, dtype=torch.int32), row_ids=t["row_ids"][:0])
    out = torch.full_like(t["q"], 2.0)
    assert (run(t, gpu, out=out) == 2.0).all()
    assert (run(t, gpu, out=out, max_chunk=None) == 2.0).all()


def _lengths(seed, B, most, far):
    """B chunks of up to `most` tokens, two empty, behind contexts of very unequal lengths."""
    g = torch.Generator().manual_seed(seed)
    chunks = torch.randint(1, most + 1, (B,), generator=g)
    chunks[0], chunks[B // 2], chunks[-1] = most, 0, 0
    ctxs = (torch.rand(B, generator=g) ** 4 * far).int()
    return chunks.tolist(), ctxs.tolist()


@pytest.mark.parametrize("B,most,far,hq,hkv,bs", [
    (24, 600, 5000, 32, 8, 16),     # eight waves, a few items a workgroup
    (100, 30, 3000, 32, 8, 16),     # four waves
    (60, 150, 900, 40, 5, 32),      # KV heads that no round divides by
    (256, 20, 200, 32, 2, 16),      # two KV heads, as many sequences as are tabulated
    (90, 200, 1, 16, 2, 16),        # prompts
    (257, 20, 200, 16, 8, 16),      # one sequence more: items in order
    (25, 800, 1, 16, 1, 16),        # few sequences of one KV head
    (40, 1000, 1, 16, 1, 16),       # more row tiles than are tabulated
])
def test_more_items_than_workgroups(gpu, B, most, far, hq, hkv, bs):
    announce(f"{B} chunks of up to {most}, contexts up to {far}, heads {hq}/{hkv}")
    t = make_case(*_lengths(B, B, most, far), hq, hkv, bs, gpu, seed=B, tail=3)
    t["row_ids"][1] = -1  # no row of the table: zeros
    out = torch.full_like(t["q"], 7.0)
    run(t, gpu, out=out)
    torch.cuda.synchronize()
    check(out, t, f"{B} chunks")
    assert (out[-3:] == 7.0).all()
    again = run(t, gpu)
    assert torch.equal(again[:-3], out[:-3]), "the same call gave other bits"


def test_many_items_of_one_length(gpu):
    announce("chunk: 64 chunks of 64 tokens behind 100 each")
    t = make_case([64] * 64, [100] * 64, 32, 8, 16, gpu, seed=14)
    check(run(t, gpu), t, "one length")


def test_replay_of_many_items_with_other_lengths(gpu):
    announce("chunk: many items, captured and replayed with other lengths")
    t = make_case(*_lengths(15, 30, 300, 2000), 32, 8, 16, gpu, seed=15)
    dev = {k: t[k].to(gpu) for k in ("table", "seq_lens", "row_ids", "cu")}
    from qwen3_engine_from_scratch_amd.kernels.paged_attention import paged_attention_chunk_hip

    out = torch.empty_like(t["q"])

    def call():
        paged_attention_chunk_hip(t["q"], t["k"], t["v"], dev["table"], dev["seq_lens"],
                                  dev["row_ids"], dev["cu"], 16, max_chunk=t["most"], out=out)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(3):
        for b in range(i, 30, 3):
            r = int(t["row_ids"][b])
            t["seq_lens"][r] = int(t["seq_lens"][r]) // 2
        dev["seq_lens"].copy_(t["seq_lens"])
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        check(out, t, f"replay {i}")
