"""Decode attention over shared prefixes with groups' bounds that do not ascend: groups that
would overlap are none."""
import pytest
import torch

from conftest import announce
from test_shared_gpu import check, make_shared, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,hq", [(4, 16), (40, 32), (600, 16)])
def test_groups_that_overlap(gpu, n, hq):
    announce(f"shared: {n} sequences in groups that overlap")
    t = make_shared([(320, [1 + i % 50 for i in range(n)])], hq, 8, 16, gpu, seed=n)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    t["groups"], t["shared"] = i32([0]), i32([])
    alone = run(t, gpu)
    check(alone, t, "alone")
    many = [0, n] * (n // 2)
    for cu, shared in (([0, n, 0, n], [320, 0, 64]), ([n // 2, n, 0], [320, 320]), ([0, n, n - 1], [320, 5]),
                       (many, [320 - 16 * (i % 7) for i in range(len(many) - 1)]),
                       ([0, n, -5], [320, 0]), ([0, 2 ** 31 - 1, n], [320, 320])):
        t["groups"], t["shared"] = i32(cu), i32(shared)
        out = run(t, gpu)
        torch.cuda.synchronize()
        check(out, t, f"bounds {cu[:4]}")
        assert torch.equal(out, alone), f"bounds {cu[:4]}"
    t["groups"], t["shared"] = i32([0, n]), i32([320])  # (and ascending ones are groups)
    assert not torch.equal(run(t, gpu), alone)
