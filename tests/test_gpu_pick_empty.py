"""Histories without a place: an empty context, as a first step has one."""
import pytest
import torch

from test_gpu_draft import Logits, i32

pytestmark = pytest.mark.gpu

CALLS = [([1, 5, 3], 1000), ([3, 2], 262149)]       # a small call, and a large one


def empties(B):
    return (torch.zeros(B, 0, dtype=torch.int32, device="cuda"),
            torch.ones(B, 9, dtype=torch.int32, device="cuda")[:, :0])


@pytest.mark.parametrize("sizes, V", CALLS)
@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("tree", [False, True])
def test_history_without_places(cuda, sizes, V, form, tree):
    c = Logits(sizes, V, torch.float32, seed=4, bias="all", tree=tree, history=0)
    c.kw["history"] = empties(len(sizes))[form]
    assert c.kw["history"].shape[1] == 0 and not c.kw["history_len"].any()
    c.check()


@pytest.mark.parametrize("sizes, V", CALLS)
def test_history_longer_than_its_places(cuda, sizes, V):
    """Counted as none, and said."""
    from warp_b200 import ffi, ops
    ops.attn_status()
    x = torch.randn(sum(sizes), V, generator=torch.Generator().manual_seed(5)).cuda()
    q_start = i32([0] + sizes).cumsum(0).int().cuda()
    picked = ops.pick_tokens(x, q_start, max_q=max(sizes), history=empties(len(sizes))[0],
                             history_len=i32([0] * (len(sizes) - 1) + [3]).cuda(),
                             presence=torch.full((len(sizes),), 9.0, device="cuda"))
    with pytest.raises(ffi.WarpError, match="length"):
        ops.attn_status()
    assert picked.tolist() == x.argmax(1).tolist()
