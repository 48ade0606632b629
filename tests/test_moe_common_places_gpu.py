"""Grouped products whose offsets do not ascend and give places to several groups: the call ends, writes results of a place's own groups or nothing, and
leaves every other row as it was."""
import pytest
import torch

import moeref
from brain_amd import ops
from test_moe_ops_gpu import gen, operands

pytestmark = pytest.mark.gpu

# Few rows; rows enough for tiles of 64 and of 128; for tiles of 256 (by the rows an expert, and the tiles that there may be).
STEP = [0, 16] * 20 + [17]
CASES = [(17, STEP, 96, 64), (17, STEP, 30, 60), (17, STEP, 300, 128), (310, [0, 300] * 6 + [0, 310], 700, 256), (310, [0, 300] * 6 + [0, 310], 700, 260),
         (40000, [0, 20000, 0, 20100, 30, 40000], 700, 128), (700, [700, 0] * 300 + [5, 90], 300, 128)]


@pytest.mark.parametrize("places,offsets,n,k", CASES)
def test_common_places(gpu, places, offsets, n, k):
    experts = len(offsets) - 1
    xq, wq, sx, sw, _ = operands(50, experts, n, k, places, gpu)
    rows = torch.randint(0, 50, (places,), generator=gen(places), dtype=torch.int32).to(gpu)
    at = torch.tensor(offsets, dtype=torch.int32, device=gpu)
    left = -2 ** 31  # no sum is
    out = torch.full((places, n), left, dtype=torch.int32, device=gpu)
    ops.matmul_i8_grouped(xq, wq, sx, sw, at, rows, out=out)
    x = xq.cpu().view(torch.int8).double()[rows.cpu().long()]
    ok = out.cpu() == left
    used, first = torch.zeros(places, dtype=torch.bool), True
    for e in range(experts):
        a, b = offsets[e], offsets[e + 1]
        if a >= b:
            continue
        acc = (x[a:b] @ wq[e].cpu().view(torch.int8).double().t()).to(torch.int32)
        if first:
            assert bool((out[a:b] != left).all())  # the first group's rows are results of some group
        first, used[a:b] = False, True
        ok[a:b] |= out[a:b].cpu() == acc
    assert bool(ok.all())
    assert bool((out.cpu()[~used] == left).all())
