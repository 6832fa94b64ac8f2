"""Pages that lie beyond 2^31 elements (and 2^32 bytes) of the pool."""
import pytest
import torch

from conftest import announce
from test_chunk_gpu import check, make_case, run

pytestmark = pytest.mark.gpu

BLOCKS, LAYERS, HEADS, BS, D = 5000, 28, 8, 16, 128


@pytest.fixture(scope="module")
def pools(gpu):
    big = [torch.empty(BLOCKS, LAYERS, HEADS, BS, D, dtype=torch.bfloat16, device=gpu)
           for _ in range(2)]
    assert big[0].numel() > 1 << 31
    yield big
    big.clear()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("chunks,ctxs", [([4, 1], [300, 40]),          # few rows
                                         ([70, 5], [300, 40]),         # ranges
                                         ([60] * 40, [100] * 40)])     # dealt
def test_chunk(gpu, pools, chunks, ctxs):
    announce(f"chunk {chunks[:3]}: the last blocks of a pool of {BLOCKS}")
    t = make_case(chunks, ctxs, 32, HEADS, BS, gpu, seed=3)
    blocks = t["k"].shape[0]
    for big, name in zip(pools, ("k", "v")):
        big[BLOCKS - blocks:, LAYERS - 1] = t[name]
    moved = dict(t, k=pools[0][:, LAYERS - 1], v=pools[1][:, LAYERS - 1],
                 table=torch.where(t["table"] >= 0, t["table"] + (BLOCKS - blocks), -1))
    out = run(moved, gpu)
    torch.cuda.synchronize()
    check(out, t, "far blocks")


def test_pages_and_rotary(gpu, pools):
    from qwen3_engine_from_scratch_amd.kernels.paged_cache import (copy_pages_hip, fork_pages_hip,
                                                                  move_pages_hip)
    from qwen3_engine_from_scratch_amd.kernels.rotary import (make_rotary, rotary_embedding_hip,
                                                             rotary_embedding_prefill_hip)

    announce("copies, forks, moves and rotated keys in the last blocks")
    far = BLOCKS - 1
    g = torch.Generator(device=gpu).manual_seed(1)
    for big in pools:
        big[:3].normal_(generator=g)
        big[far - 3:] = 0
    copy_pages_hip(*pools, [0], [far])
    for big in pools:
        assert torch.equal(big[far], big[0])
    table = torch.full((3, 4), -1, dtype=torch.int32, device=gpu)
    table[0, 0] = far
    lens = torch.zeros(3, dtype=torch.int32, device=gpu)
    fork_pages_hip(*pools, table, lens, [0], [1], [5], [far - 1])
    assert table[1].tolist() == [far - 1, -1, -1, -1] and lens.tolist() == [0, 5, 0]
    for big in pools:
        assert torch.equal(big[far - 1][:, :, :5], big[0][:, :, :5])
        assert not big[far - 1][:, :, 5:].any()
    move_pages_hip(*pools, table, [far], [1])
    assert table[0, 0] == 1
    for big in pools:
        assert torch.equal(big[1], big[0])
    x = torch.randn(4, 24, D, generator=g, device=gpu).to(torch.bfloat16)
    q, k, v = x[:, :8], x[:, 8:16], x[:, 16:]
    pos = torch.tensor([0, 7, 100, 5], device=gpu)
    rot = make_rotary(D, device=gpu)
    slots = torch.tensor([(far - 2) * BS, (far - 2) * BS + 15, -1, (far - 3) * BS + 1], device=gpu)
    rotary_embedding_prefill_hip(q, k, v, pos, rot, slots, *pools, LAYERS - 1)
    _, kr = rotary_embedding_hip(q, k, pos, rot)
    for i, s in enumerate(slots.tolist()):
        if s >= 0:
            assert torch.equal(pools[0][s // BS, LAYERS - 1, :, s % BS], kr[i])
            assert torch.equal(pools[1][s // BS, LAYERS - 1, :, s % BS], v[i])
