"""The range of experts that bh_moe_plan_rows (ops.moe_plan) takes: up to the last int32, no further, so that no negative expert is of it."""
import pytest
import torch

import moeref
from brain_amd import load, ops
from test_kvops_validation import P, i, refused
from test_moe_ops_validation import plan


@pytest.mark.parametrize("first,n", [(2 ** 32 - 1, 1), (2 ** 32 - 1, 60), (2 ** 31 - 1, 2), (2 ** 31 - 1023, 1024), (2 ** 31, 1)])
def test_entry(first, n):
    refused(load().bh_moe_plan_rows(None, P, 5, 4, first, n, plan(), None, 0), f"first {first}", "2^31")


@pytest.mark.parametrize("first,n", [(2 ** 31 - 1, 2), (2 ** 31 - 1023, 1024), (2 ** 31, 1)])
def test_ops(first, n):
    with pytest.raises(ValueError, match=f"first {first}"):
        ops.moe_plan(i(5, 4), n, first=first)


@pytest.mark.gpu
@pytest.mark.parametrize("first,n", [(2 ** 31 - 1, 1), (2 ** 31 - 8, 8), (2 ** 31 - 1024, 1024), (0, 3)])
@pytest.mark.parametrize("tokens", [4, 3000])
def test_last_range(gpu, first, n, tokens):
    """The last experts that there are, beside negative ones of every distance."""
    e = torch.randint(first, min(first + n, 2 ** 31 - 1) + 1, (tokens, 4), generator=torch.Generator().manual_seed(n)).clamp_max(2 ** 31 - 1)
    e[1::3] -= 2 ** 31  # negative
    e[2::3] = torch.tensor([-1, -2 ** 31, 2 ** 31 - 1, -2 ** 31 + 1])
    got = ops.moe_plan(e.to(torch.int32).to(gpu), n, first=first)
    offsets, rows, slots = moeref.plan(e.numpy(), n, first)
    assert got.offsets.tolist() == offsets.tolist()
    assert got.rows[: len(rows)].tolist() == rows.tolist()
    assert got.slots.tolist() == slots.tolist()
