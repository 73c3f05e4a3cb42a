"""Operators on drafted tokens where offsets pass 32 bits, and calls that run at once."""
import pytest
import torch

from test_gpu_draft import RAGGED, Drafted, Logits, Trees, i32, starts_of, trees_of

pytestmark = pytest.mark.gpu


def far(x):
    """x on the device, its first axis so wide that the last entries lie past 2^31 elements."""
    step = (2 ** 31 // (len(x) - 1) // 16 + 1) * 16
    room = torch.empty((len(x) - 1) * step + x[0].numel(), dtype=x.dtype, device="cuda")
    y = torch.as_strided(room, x.shape, (step, *x[0].contiguous().stride()))
    assert y[-1].data_ptr() - y.data_ptr() >= 2 ** 32
    return y.copy_(x)


@pytest.mark.parametrize("q, D, runs", [(1, 64, False), (1, 128, False), (26, 64, False),
                                        (26, 128, False), (26, 128, True)])
def test_far_pages(cuda, q, D, runs):
    sizes = [min(q, k) for k in RAGGED]
    c = Trees(trees_of(sizes), RAGGED, 16, 4, D, 16, torch.bfloat16, seed=q, runs=runs)
    c.place = far
    c.check()


def test_far_paths(cuda):
    c = Drafted([26, 3, 40], 50, tokens=2, seed=2, layers=1)
    n = c.pools.shape[2]
    step = (2 ** 31 // (n - 1) // 16 + 1) * 16
    room = torch.empty(n * step, dtype=c.pools.dtype, device="cuda")
    size = c.pools[0, 0, 0].numel()
    pools = torch.as_strided(room, c.pools.shape, (2 * size, size, step, *c.pools.stride()[3:]))
    c.pools = pools.copy_(c.pools)
    c.check()


@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
def test_far_rows(cuda, large, in_place):
    Logits([5, 1, 3], 1003, torch.bfloat16, seed=6, bias="all", masked=True, large=large).check(
        place=far, in_place=in_place)


def test_calls_at_once(cuda):
    """Steps on several streams, each with tensors of its own, give what each gives alone."""
    from warp_b200 import ops
    works = []
    for seed in range(3):
        sizes = [min(20 + seed, k) for k in RAGGED]
        c = Trees(trees_of(sizes, seed=seed), RAGGED, 16, 4, 128, 16, torch.bfloat16, seed=seed,
                  runs=seed != 1)
        few, many = (Logits(sizes, 5000, torch.float32, seed=seed, large=large)
                     for large in (False, True))
        a = Drafted(sizes, 50, tokens=2, seed=seed)
        args = [x.cuda() for x in (c.q, c.k, c.v, c.pages, i32(RAGGED), i32(starts_of(sizes)),
                                   c.seen)]
        picks = [(x.x.cuda(), {k: v.cuda() if torch.is_tensor(v) else v for k, v in x.kw.items()})
                 for x in (few, many)]
        check = [x.cuda() for x in (i32(a.drafted), i32(a.picked), a.seen, i32(starts_of(sizes)),
                                    i32(a.kv))]
        parents = i32([p for t in a.trees for p in t]).cuda()
        wide = a.pages.shape[1]

        def work(c=c, args=args, picks=picks, check=check, a=a, parents=parents, wide=wide,
                 n=max(sizes), T=sum(sizes)):
            pages = torch.full((len(RAGGED), wide), -1, dtype=torch.int32, device="cuda")
            held = torch.zeros(len(RAGGED), dtype=torch.int32, device="cuda")
            plan = ops.step_plan(check[3], check[4], pages, 16, T, held=held, max_q=n,
                                 pool=ops.page_pool(len(RAGGED) * wide), parents=parents)
            return [*plan, pages, ops.tree_attention(*args, n, c.max_kv),
                    *(ops.pick_tokens(x, **kw) for x, kw in picks),
                    *ops.tree_accept(*check, n)]
        works.append(work)
    alone = [work() for work in works]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in works]
    for _ in range(5):
        got = []
        for stream, work in zip(streams, works):
            with torch.cuda.stream(stream):
                got.append(work())
        torch.cuda.synchronize()
        for one, want in zip(got, alone):
            assert len(one) == len(want) and all(torch.equal(x, y) for x, y in zip(one, want))
    ops.attn_status()
