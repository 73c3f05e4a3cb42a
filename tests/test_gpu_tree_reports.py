"""Tree attention whose blocks take equal runs reports a broken request as the other ways
do, also one that is left without a row or a key."""
import pytest
import torch

from test_gpu_draft import Trees, i32, trees_of

pytestmark = pytest.mark.gpu

KV = [700, 40, 300, 90]
SIZES = [9, 5, 12, 3]
STARTS = [0, 9, 14, 26, 29]


@pytest.mark.parametrize("kv, starts, rows", [
    ([700, -4, 300, 90], STARTS, {1: "none"}),              # a length below zero
    ([700, 40, 300, -1], STARTS, {3: "none"}),
    (KV, [0, 9, 14, 26, 31], {}),                           # an end past the tokens
    ([700, 40, 0, 90], [0, 9, 14, 33, 36], {2: "none", 3: None}),   # a request past them
    (KV, [9, 9, 7, 19, 22], {0: None, 1: None, 2: "other", 3: "other"}),    # starts that descend
    ([700, 0, 300, 90], [0, 1, 14, 26, 29], {0: "other", 1: "none"}),   # nodes past the bound, no key
])
@pytest.mark.parametrize("runs", [False, True])
def test_broken_requests_are_reported(cuda, runs, kv, starts, rows):
    """`rows`: requests that have no row now (None), zeros (without a key) or other rows than
    before; all others have what they had."""
    from warp_b200 import ffi, ops
    c = Trees(trees_of(SIZES), KV, 16, 4, 64, 16, torch.bfloat16, seed=3, runs=runs)
    good = c.run()
    out = torch.full_like(c.q, 7.0).cuda()
    ops.tree_attention(c.q.cuda(), c.k.cuda(), c.v.cuda(), c.pages.cuda(), i32(kv).cuda(),
                       i32(starts).cuda(), c.seen.cuda(), c.max_q, c.max_kv, out=out)
    with pytest.raises(ffi.WarpError, match="length"):
        ops.attn_status()
    ops.attn_status()
    for b, n in enumerate(SIZES):
        mine = out[STARTS[b]:STARTS[b] + n].cpu()
        if b not in rows:
            assert torch.equal(mine, good[STARTS[b]:STARTS[b] + n])
        elif rows[b] == "none":
            t0 = starts[b]
            assert not out[t0:min(t0 + c.max_q, starts[b + 1])].any()


@pytest.mark.parametrize("kv, sizes", [([700, 0, 300, 0], [9, 5, 0, 0]), ([0, 0], [0, 3])])
def test_requests_without_keys_or_nodes_are_none(cuda, kv, sizes):
    """They are no fault."""
    c = Trees(trees_of(sizes + [9]), kv + [50], 16, 4, 64, 16, torch.bfloat16, seed=4, runs=True)
    c.check()
