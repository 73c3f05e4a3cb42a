"""A pool that runs empty, over a page table whose entries were never set: keys without a page
have no slot, and no other request's page stands for theirs."""
import pytest
import torch

from test_gpu_draft import i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("junk", [0, 3, 1 << 30])
@pytest.mark.parametrize("batch, tokens", [(3, 1), (3, 400), (1500, 1)])
def test_entries_without_a_page(cuda, junk, batch, tokens):
    """The last requests lack pages; the table holds numbers of pages that others have."""
    from warp_b200 import ffi, ops
    ops.attn_status()
    page, wide, n = 16, 40, batch * 30 + 2
    kv = 630                                # 40 pages each
    pages = torch.full((batch, wide), junk, dtype=torch.int32, device="cuda")
    held = torch.zeros(batch, dtype=torch.int32, device="cuda")
    pool = ops.page_pool(n)
    q_start = (torch.arange(batch + 1) * tokens).int().cuda()
    T = batch * tokens
    _, slots = ops.step_plan(q_start, torch.full((batch,), kv, dtype=torch.int32, device="cuda"),
                             pages, page, T, held=held, pool=pool)
    with pytest.raises(ffi.WarpError, match="no page left"):
        ops.attn_status()
    want = torch.arange(batch * wide).view(batch, wide)
    want[want >= n] = -1
    assert torch.equal(pages.cpu(), want.int()) and pool[0] == 0
    assert torch.equal(held.cpu(), (want >= 0).sum(1).int())
    j = torch.arange(kv - tokens, kv)
    at = want[:, j // page]
    assert torch.equal(slots.cpu(), torch.where(at >= 0, at * page + j % page, -1).flatten())


def test_a_short_pool_leaves_the_rest_of_the_table(cuda):
    """Entries past what a request needs, and those of requests that lack nothing, stay."""
    from warp_b200 import ffi, ops
    ops.attn_status()
    pages = torch.full((3, 6), 9, dtype=torch.int32, device="cuda")
    held = i32([0, 1, 0]).cuda()
    pool = ops.page_pool(3)
    ops.step_plan(i32([0] * 4).cuda(), i32([20, 40, 64]).cuda(), pages, 16, 0, held=held, pool=pool)
    with pytest.raises(ffi.WarpError, match="no page left"):
        ops.attn_status()
    assert pages.tolist() == [[0, 1, 9, 9, 9, 9], [9, 2, -1, 9, 9, 9], [-1] * 4 + [9, 9]]
    assert held.tolist() == [2, 2, 0]


def test_moves_stay_within_the_pages_held(cuda):
    """An accepted path of a request that lacks pages moves nothing into another's."""
    from warp_b200 import ffi, ops
    ops.attn_status()
    page, n = 16, 10
    pages = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    held, pool = i32([0, 0]).cuda(), ops.page_pool(3)
    q_start, kv = i32([0, 0, n]).cuda(), i32([32, 24]).cuda()
    parents = i32([-1, 0, 0, 1, 2, 3, 4, 6, 7, 8]).cuda()
    _, _, seen = ops.step_plan(q_start, kv, pages, page, n, held=held, pool=pool, parents=parents,
                               max_q=n)
    assert held.tolist() == [2, 1]
    k, v = (torch.randn(1, 4, page, 1, 64, generator=torch.Generator().manual_seed(i)).half().cuda()
            for i in range(2))
    kept = k[0, [0, 1, 3]].clone(), v[0, [0, 1, 3]].clone()
    tokens = torch.ones(n, dtype=torch.int32, device="cuda")
    count = ops.tree_accept(tokens, tokens, seen, q_start, kv, n, caches=(k, v), pages=pages)[0]
    with pytest.raises(ffi.WarpError, match="no page left"):
        ops.attn_status()
    assert count.tolist() == [0, 7]
    assert torch.equal(k[0, [0, 1, 3]], kept[0]) and torch.equal(v[0, [0, 1, 3]], kept[1])
