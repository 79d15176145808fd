"""What a packed plan takes for its host integers; CPU only."""

import numpy as np
import pytest
import torch

from torch2iron_amd import ops


@pytest.mark.parametrize("bad", [2.9, 2.0, np.float32(2), torch.tensor(2.5), "2", None],
                         ids=["fraction", "float", "numpy", "tensor", "text", "none"])
def test_what_is_no_integer_is_refused(bad):
    """Not cut to one: 2.9 rows are not 2."""
    for kw in (dict(lengths=[bad, 1]), dict(lengths=[1, 1], starts=[0, bad]), dict(lengths=[1, 1], cache_rows=[0, bad])):
        with pytest.raises(ValueError, match="integers"):
            ops.PackedPlan(kw.pop("lengths"), 4, 2, 16, "cpu", **kw)


@pytest.mark.parametrize("make", [list, tuple, np.array, torch.tensor, lambda v: torch.tensor(v, dtype=torch.int32),
                                  lambda v: [np.int64(x) for x in v]])
def test_integers_of_any_kind(make):
    plan = ops.PackedPlan(make([3, 0, 2]), 4, 2, 16, "cpu", starts=make([1, 2, 3]), cache_rows=make([2, 0, 1]))
    assert (plan.lengths, plan.starts, plan.cache_rows, plan.rows) == ([3, 0, 2], [1, 2, 3], [2, 0, 1], 5)
    assert all(type(x) is int for x in plan.lengths + plan.starts + plan.cache_rows)


def test_plan_under_another_default_device():
    """The plan is made in host memory whatever torch's default device: its entry point reads and writes it there
    (a tensor on the default device has no host address)."""
    want = ops.PackedPlan([40, 0, 3], 4, 2, 512, "cpu", starts=[0, 0, 500])
    with torch.device("meta"):
        plan = ops.PackedPlan([40, 0, 3], 4, 2, 512, "cpu", starts=[0, 0, 500])
    assert plan.table.device.type == "cpu" and torch.equal(plan.table, want.table)
