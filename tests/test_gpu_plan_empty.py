"""A plan of no request leaves the pool as it is."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_plan_of_an_empty_batch(cuda):
    from warp_b200 import ops
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    pool = ops.page_pool(5)
    for kw in ({}, dict(held=none, pool=pool)):
        positions, slots = ops.step_plan(torch.zeros(1, dtype=torch.int32, device="cuda"), none,
                                         none.view(0, 4), 16, 0, **kw)
        assert positions.shape == slots.shape == (0,)
    ops.attn_status()
    assert pool.tolist() == [5, 4, 3, 2, 1, 0]
