"""Rows a request of a pick: all of them where no bound is given, -1 for those past one,
nothing for rows of no request; and contexts without a place."""
import pytest
import torch

from test_gpu_draft import Logits, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sizes, tree", [([5, 0, 70, 1, 3], True), ([5, 0, 70, 1, 3], False),
                                         ([1, 1], True), ([64], True), ([200, 7], True)])
def test_every_row_without_a_bound(cuda, dtype, sizes, tree, large):
    """Requests bring what q_start says, whether or not there are masks."""
    c = Logits(sizes, 1000, dtype, seed=len(sizes), masked=True, tree=tree, large=large)
    del c.kw["max_q"]
    c.check()


def test_a_workload_without_a_bound(cuda):
    """Trees of unequal size over a large vocabulary, on the way of large calls by it alone."""
    c = Logits([26, 5, 13, 1, 20], 100003, torch.bfloat16, seed=3, masked=True, history=900)
    del c.kw["max_q"]
    c.check()


def raw(x, q_start, max_q, out, wide=0):
    """warp_pick_tokens over results that were there: `wide` places of an empty history
    make it a large call."""
    from warp_b200 import ffi, ops
    T, V = x.shape
    B = q_start.numel() - 1
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    history = torch.zeros(B, wide, dtype=torch.int32, device="cuda") if wide else None
    picked = torch.full((T,), 7, dtype=torch.int32, device="cuda")
    d = ffi.PICK_DESC.pack(T, B, V, ops._TYPES[x.dtype], max_q, x.data_ptr(), V, out.data_ptr(), V,
                           picked.data_ptr(), q_start.data_ptr(), history.data_ptr() if wide else 0,
                           lens.data_ptr() if wide else 0, wide, wide, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    lib = ffi.load()
    need = lib.warp_pick_scratch(d)
    assert (need > 0) == bool(wide)
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    ffi.check(lib.warp_pick_tokens(d, scratch.data_ptr() if need else None, ops._stream()))
    return picked


@pytest.mark.parametrize("wide", [0, 16400])
def test_rows_past_the_bound_are_minus_one(cuda, wide):
    """Of three requests' 4, 2 and 5 rows two are taken; rows of no request stay as they were."""
    from warp_b200 import ffi, ops
    ops.attn_status()
    x = torch.randn(14, 9000, generator=torch.Generator().manual_seed(1)).cuda()
    out = torch.full_like(x, 5.0)
    picked = raw(x, i32([1, 5, 7, 12]).cuda(), 2, out, wide)
    with pytest.raises(ffi.WarpError, match="length"):
        ops.attn_status()
    top = x.argmax(1).tolist()
    assert picked.tolist() == [7] + top[1:3] + [-1] * 2 + top[5:9] + [-1] * 3 + [7] * 2
    taken = [1, 2, 5, 6, 7, 8]
    assert torch.equal(out[taken], x[taken])
    assert (out[[t for t in range(14) if t not in taken]] == 5).all()


@pytest.mark.parametrize("wide", [0, 16400])
def test_a_start_before_the_rows_is_minus_one(cuda, wide):
    from warp_b200 import ffi, ops
    ops.attn_status()
    x = torch.randn(5, 9000, generator=torch.Generator().manual_seed(2)).cuda()
    picked = raw(x, i32([-1, 2, 4]).cuda(), 9, torch.full_like(x, 5.0), wide)
    with pytest.raises(ffi.WarpError, match="length"):
        ops.attn_status()
    assert picked.tolist() == [-1] * 2 + x[2:4].argmax(1).tolist() + [7]


def test_masks_are_the_bound_without_another(cuda):
    """A row of masks holds 64 nodes; a request with more has no choice behind them."""
    from warp_b200 import ffi, ops
    ops.attn_status()
    x = torch.randn(70, 300, generator=torch.Generator().manual_seed(3)).cuda()
    seen = torch.ones(70, 1, dtype=torch.int64, device="cuda")
    drafted = torch.zeros(70, dtype=torch.int32, device="cuda")
    picked = ops.pick_tokens(x, i32([0, 70]).cuda(), drafted=drafted, seen=seen)
    with pytest.raises(ffi.WarpError, match="length"):
        ops.attn_status()
    assert picked.tolist() == x[:64].argmax(1).tolist() + [-1] * 6


def test_a_bound_of_no_row(cuda):
    from warp_b200 import ops
    x = torch.randn(3, 50).cuda()
    for starts in ([0, 3], [0, 0]):
        assert ops.pick_tokens(x, i32(starts).cuda(), max_q=0).tolist() == [-1] * 3
    assert ops.pick_tokens(x[:0], i32([0, 0]).cuda()).shape == (0,)
