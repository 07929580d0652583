"""The layout of a prefill batch's keys over the 4-bit KV cache: what it holds and how much."""

import pytest
import torch

from minisgl import ops

CPU = torch.device("cpu")


def _tensors(plan):
    return [x for x in vars(plan).values() if isinstance(x, torch.Tensor)]


@pytest.mark.parametrize("lens", [[131072] + [40] * 1000, [40] * 1279, [1], [5000, 1, 1]], ids=["long", "many", "one", "few"])
def test_a_plan_takes_some_bytes_a_key(lens):
    """Two numbers a key, in whole tiles, and one a request: not the requests times the longest."""
    plan = ops.KV4PrefillPlan(lens, CPU)
    rows = sum(-(-n // 128) * 128 for n in lens)
    held = {x.untyped_storage().data_ptr(): x.untyped_storage().nbytes() for x in _tensors(plan)}
    assert sum(held.values()) <= 4 * (2 * rows + len(lens) + 1)


@pytest.mark.parametrize("lens", [[300, 0, 128, 1], [0, 0], [129], [-5, 3]])
def test_rows_of_a_plan(lens):
    plan = ops.KV4PrefillPlan(lens, CPU)
    at = 0
    for b, n in enumerate(lens):
        tiles = -(-max(n, 0) // 128)
        assert plan.first_row[b] == at
        assert plan.row_req[at:at + tiles * 128].tolist() == [b] * max(n, 0) + [-1] * (tiles * 128 - max(n, 0))
        assert plan.row_pos[at:at + max(n, 0)].tolist() == list(range(max(n, 0)))
        at += tiles * 128
    assert plan.rows == at == plan.row_req.numel() == plan.row_pos.numel()
    assert all(x.dtype == torch.int32 and x.is_contiguous() for x in _tensors(plan))


def test_a_plan_of_no_requests():
    plan = ops.KV4PrefillPlan([], CPU)
    assert plan.rows == 0 and all(x.numel() == 0 for x in _tensors(plan))
