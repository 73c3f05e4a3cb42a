"""A step's plan refuses lengths that its pages or its tokens cannot have."""
import pytest
import torch

from warp_b200 import ops
from warp_b200.block import Step


class Planned(Exception):
    pass


@pytest.fixture(autouse=True)
def no_device(monkeypatch):
    def kv_slots(*a, **kw):
        raise Planned
    monkeypatch.setattr(ops, "kv_slots", kv_slots)


def table(batch, n):
    return torch.zeros(batch, n, dtype=torch.int32)


@pytest.mark.parametrize("q, kv, n", [([1, 1], [33, 5], 2), ([3], [2], 1), ([1], [0], 4),
                                      ([-1], [4], 1), ([1, 0, 2], [1, 0, 65], 4), ([1], [1], 0)])
def test_lengths_that_do_not_fit(q, kv, n):
    with pytest.raises(ValueError, match="request"):
        Step.plan(q, kv, table(len(q), n), 16)


def test_rows_of_pages_for_each_request():
    with pytest.raises(ValueError, match="request"):
        Step.plan([1, 1], [1, 1], table(1, 4), 16)


@pytest.mark.parametrize("pages, n", [(None, 1), (2, 33), (0, 1), (2, -1)])
def test_prefix_that_its_pages_do_not_hold(pages, n):
    front = None if pages is None else table(1, pages)[0]
    with pytest.raises(ValueError, match="prefix"):
        Step.plan([1], [1], table(1, 1), 16, prefix_pages=front, prefix_len=n)


@pytest.mark.parametrize("q, kv, n", [([1, 0], [32, 0], 2), ([16], [16], 1), ([0], [16], 1)])
def test_lengths_that_fit(q, kv, n):
    with pytest.raises(Planned):
        Step.plan(q, kv, table(len(q), n), 16)
    with pytest.raises(Planned):
        Step.plan(q, kv, table(len(q), n), 16, prefix_pages=table(1, 2)[0], prefix_len=32)
