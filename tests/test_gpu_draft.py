"""A step of drafted tokens against plain implementations: the plan and the check
of drafted tokens exactly, adjusted logits bit for bit against the same fp32
operations, tree attention against 64 bits.

Tolerance of the attention: u is the type's unit roundoff (2^-8 bf16 and 2^-11 fp16, half
of torch.finfo(t).eps).  The weights are rounded to the type before the second
product, which moves a result by at most u * sum p|v| / l, and the result is
rounded once, u |o|.  A score is an fp32 sum of D products of magnitude below some
40 in all, off by at most 2^-15, and the exponential by 2^-13.7: together less than
2^-13 of each weight, in numerator and denominator alike, 2^-12 of sum p|v| / l.
"""
import math
import random

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def starts_of(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def random_parents(rng, n, kind):
    if kind == "chain":
        return [-1] + list(range(n - 1))
    if kind == "star":
        return [-1] + [0] * (n - 1)
    if kind == "forest":                    # several roots
        return [-1] + [rng.choice([-1, rng.randrange(i)]) for i in range(1, n)]
    return [-1] + [rng.randrange(max(0, i - 6), i) for i in range(1, n)]


def paths_of(parents):
    paths = []
    for i, p in enumerate(parents):
        paths.append((paths[p] if p >= 0 else []) + [i])
    return paths


def words_of(paths, words):
    rows = []
    for p in paths:
        bits = sum(1 << m for m in p)
        rows.append([(bits >> 64 * w & (1 << 64) - 1) for w in range(words)])
    return [[x - (1 << 64) if x >> 63 else x for x in row] for row in rows]


def seen_of(trees, max_q):
    words = -(-max_q // 64)
    rows = [row for parents in trees for row in words_of(paths_of(parents), words)]
    return torch.tensor(rows, dtype=torch.int64).view(-1, words)


# ---- plan ----------------------------------------------------------------------------


class Book:
    """The page table and the pool as lists, page by page."""

    def __init__(self, batch, wide, n, page):
        self.rows = [[] for _ in range(batch)]
        self.free, self.wide, self.page, self.n = list(range(n - 1, -1, -1)), wide, page, n

    def to(self, lengths):
        need = [min(-(-max(0, n) // self.page), self.wide) for n in lengths]
        for row, k in reversed(list(zip(self.rows, need))):
            while len(row) > k:
                self.free.append(row.pop())
        for row, k in zip(self.rows, need):
            while len(row) < k and self.free:
                row.append(self.free.pop())

    def table(self):
        return i32([r + [-1] * (self.wide - len(r)) for r in self.rows])

    def slot(self, b, j):
        if j < 0 or j // self.page >= len(self.rows[b]):
            return -1
        return self.rows[b][j // self.page] * self.page + j % self.page


def same_state(book, pages, held, pool):
    assert torch.equal(pages.cpu(), book.table())
    assert held.tolist() == [len(r) for r in book.rows]
    got = pool.tolist()
    assert got[0] == len(book.free) and got[1:1 + got[0]] == book.free


@pytest.mark.parametrize("batch, wide, page, most", [
    (1, 9, 16, 140), (5, 40, 16, 640), (33, 6, 128, 700), (1024, 5, 16, 80), (1025, 4, 16, 64),
    (2500, 3, 32, 96)])
def test_pages_over_many_steps(cuda, batch, wide, page, most):
    """Lengths that grow, shrink and end, over a pool that just holds them."""
    from warp_b200 import ops
    rng = random.Random(batch)
    n = batch * wide
    book = Book(batch, wide, n, page)
    pages = torch.full((batch, wide), -1, dtype=torch.int32, device="cuda")
    held = torch.zeros(batch, dtype=torch.int32, device="cuda")
    pool = ops.page_pool(n)
    for step in range(6):
        kv = [rng.choice([0, 1, page, page + 1, most, rng.randint(0, most)]) for _ in range(batch)]
        if step == 4:
            kv = [0] * batch
        q = [rng.randint(0, min(k, 40)) for k in kv]
        q_start = starts_of(q)
        pos, slots = ops.step_plan(i32(q_start).cuda(), i32(kv).cuda(), pages, page, q_start[-1],
                                   base=7, held=held, pool=pool)
        book.to(kv)
        same_state(book, pages, held, pool)
        want = [(b, k - m + i) for b, (m, k) in enumerate(zip(q, kv)) for i in range(m)]
        assert pos.tolist() == [7 + j for _, j in want]
        assert slots.tolist() == [book.slot(b, j) for b, j in want]
    ops.attn_status()


def test_pages_come_back_in_order(cuda):
    """A request that shrinks and grows again has its pages again."""
    from warp_b200 import ops
    pages = torch.full((3, 8), -1, dtype=torch.int32, device="cuda")
    held = torch.zeros(3, dtype=torch.int32, device="cuda")
    pool = ops.page_pool(24)
    none = torch.zeros(4, dtype=torch.int32, device="cuda")

    def to(*kv):
        ops.step_plan(none, i32(kv).cuda(), pages, 16, 0, held=held, pool=pool)
        return pages.tolist(), pool[:1 + int(pool[0])].tolist()
    first = to(100, 30, 128)
    assert to(20, 30, 17) != first
    assert to(100, 30, 128) == first


def test_pool_runs_empty(cuda):
    from warp_b200 import ffi, ops
    ops.attn_status()
    pages = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
    held = torch.zeros(3, dtype=torch.int32, device="cuda")
    pool = ops.page_pool(5)
    q_start = i32([0, 1, 2, 3]).cuda()
    _, slots = ops.step_plan(q_start, i32([40, 50, 1]).cuda(), pages, 16, 3, held=held, pool=pool)
    assert held.tolist() == [3, 2, 0] and pool[0].item() == 0
    assert pages.tolist() == [[0, 1, 2, -1], [3, 4, -1, -1], [-1] * 4]
    assert slots.tolist() == [2 * 16 + 7, -1, -1]
    with pytest.raises(ffi.WarpError, match="no page left"):
        ops.attn_status()
    # the first request ends, and the others get what they lack
    _, slots = ops.step_plan(q_start, i32([0, 50, 1]).cuda(), pages, 16, 3, held=held, pool=pool)
    assert held.tolist() == [0, 4, 1] and pool[0].item() == 0
    assert pages.tolist() == [[-1] * 4, [3, 4, 0, 1], [2, -1, -1, -1]]
    assert slots.tolist() == [-1, 1 * 16 + 1, 2 * 16]
    ops.attn_status()


@pytest.mark.parametrize("kv, held0, count, text", [
    ([200, 3], [0, 0], 6, "length"),        # more pages than a row has
    ([-4, 3], [0, 0], 6, "length"), ([0, 3], [9, 0], 6, "page number|length"),
    ([0, 3], [-2, 0], 6, "length"), ([1, 3], [0, 0], 77, "page number"),
    ([1, 3], [0, 0], -3, "page"), ([0, 0], [4, 4], 6, "page number")])     # given back twice
def test_plan_of_broken_state(cuda, kv, held0, count, text):
    """Nothing outside the row, the pool and held is touched, and it is said."""
    from warp_b200 import ffi, ops
    ops.attn_status()
    room = torch.full((2, 8), 3, dtype=torch.int32, device="cuda")
    pages = room[:, 2:6]
    around = torch.full((40,), 5, dtype=torch.int32, device="cuda")
    pool = around[10:17]
    pool.copy_(i32([count, 0, 1, 2, 3, 4, 5]))
    held = i32(held0).cuda()
    ops.step_plan(i32([0, 0, 0]).cuda(), i32(kv).cuda(), pages, 16, 0, held=held, pool=pool)
    with pytest.raises(ffi.WarpError, match=text):
        ops.attn_status()
    assert (room[:, :2] == 3).all() and (room[:, 6:] == 3).all()
    assert (around[:10] == 5).all() and (around[17:] == 5).all()
    assert 0 <= pool[0].item() <= 6 and all(0 <= h <= 4 for h in held.tolist())


def test_plan_without_a_pool_is_kv_slots(cuda):
    from warp_b200 import ops
    q_start = i32([0, 3, 3, 4, 1200]).cuda()
    kv_len = i32([3, 50, 17, 1190]).cuda()
    pages = torch.randperm(4 * 80, dtype=torch.int32).view(4, 80).cuda()
    want = ops.kv_slots(q_start, kv_len, pages, 16, 1203, base=100)
    for a, b in zip(ops.step_plan(q_start, kv_len, pages, 16, 1203, base=100), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["chain", "star", "forest", "any"])
@pytest.mark.parametrize("sizes", [[1], [5, 0, 1, 64], [65, 2], [200, 129, 1], [30] * 50])
@pytest.mark.parametrize("pooled", [False, True])
def test_plan_of_trees(cuda, kind, sizes, pooled):
    from warp_b200 import ops
    rng = random.Random(len(sizes))
    trees = [random_parents(rng, n, kind) if n else [] for n in sizes]
    kv = [n + rng.randint(0, 50) for n in sizes]
    q_start, max_q = starts_of(sizes), max(sizes)
    batch, wide, T = len(sizes), -(-max(kv) // 16), starts_of(sizes)[-1]
    book = Book(batch, wide, batch * wide, 16)
    book.to(kv)
    kw, pages = {}, book.table().cuda()
    if pooled:
        pages.fill_(-1)
        kw = dict(held=torch.zeros(batch, dtype=torch.int32, device="cuda"),
                  pool=ops.page_pool(batch * wide))
    # two rows behind the last request
    parents = i32([p for t in trees for p in t] + [-1, 0]).cuda()
    pos, slots, seen = ops.step_plan(i32(q_start).cuda(), i32(kv).cuda(), pages, 16, T + 2, base=3,
                                     parents=parents, max_q=max_q, **kw)
    want = [(b, i, len(p) - 1) for b, t in enumerate(trees) for i, p in enumerate(paths_of(t))]
    assert pos.tolist()[:T] == [3 + kv[b] - sizes[b] + d for b, _, d in want]
    assert slots.tolist() == [book.slot(b, kv[b] - sizes[b] + i) for b, i, _ in want] + [-1, -1]
    assert torch.equal(seen.cpu()[:T], seen_of(trees, max_q)) and not seen[T:].any()
    ops.attn_status()


def test_plan_of_bad_trees(cuda):
    from warp_b200 import ffi, ops
    ops.attn_status()
    pages = torch.arange(8, dtype=torch.int32, device="cuda").view(1, 8)
    args = (i32([0, 4]).cuda(), i32([4]).cuda(), pages, 16, 4)
    for parents in ([-1, 1, 0, 2], [-1, 0, 3, 1], [0, 0, 0, 1 << 30]):
        _, _, seen = ops.step_plan(*args, parents=i32(parents).cuda(), max_q=4)
        with pytest.raises(ffi.WarpError, match="parent"):
            ops.attn_status()
        want = [-1 if p >= i else p for i, p in enumerate(parents)]
        assert torch.equal(seen.cpu(), seen_of([want], 4))
    # more nodes than the bound
    _, _, seen = ops.step_plan(*args, parents=i32([-1, 0, 1, 2]).cuda(), max_q=3)
    with pytest.raises(ffi.WarpError, match="length"):
        ops.attn_status()
    assert seen.flatten().tolist() == [1, 3, 7, 0]


@pytest.mark.parametrize("pooled", [False, True])
def test_plan_of_a_start_before_the_tokens(cuda, pooled):
    """Parents before the array are not asked for: the request's tokens have no place."""
    from warp_b200 import ffi, ops
    ops.attn_status()
    pages = torch.arange(16, dtype=torch.int32, device="cuda").view(2, 8)
    kw = dict(held=i32([8, 8]).cuda(), pool=ops.page_pool(0)) if pooled else {}
    around = torch.full((12,), 1 << 20, dtype=torch.int32, device="cuda")
    parents = around[4:10]
    parents.copy_(i32([-1, 0, 1, -1, 0, 0]))
    _, slots, seen = ops.step_plan(i32([-3, 3, 6]).cuda(), i32([128, 128]).cuda(), pages, 16, 6,
                                   parents=parents, max_q=6, **kw)
    with pytest.raises(ffi.WarpError, match="length"):
        ops.attn_status()
    assert slots.tolist() == [-1] * 3 + [8 * 16 + 125 + i for i in range(3)]
    assert seen.flatten().tolist() == [0, 0, 0, 1, 3, 5]


# ---- tree attention --------------------------------------------------------------------


class Trees:
    """Ragged requests whose queries are trees, over shuffled pages; what no request
    owns is NaN."""

    def __init__(self, trees, kv_lens, Hq, Hk, D, page, dtype, heads_first=False, prefix=0, seed=0,
                 runs=False):
        g = torch.Generator().manual_seed(seed)
        self.trees, self.kv_lens, self.prefix, self.page = trees, kv_lens, prefix, page
        self.q_lens = [len(t) for t in trees]
        B = len(trees)
        wide, front = max(1, max(-(-n // page) for n in kv_lens)), -(-prefix // page)
        total = B * wide + front + 2
        order = torch.randperm(total, generator=g).int()
        self.pages = order[:B * wide].view(B, wide).clone()
        self.pp = order[B * wide:B * wide + front].clone()
        k, v = (torch.full((total, page, Hk, D), math.nan) for _ in range(2))

        def fill(table, n):
            j = torch.arange(n)
            for x in (k, v):
                x[table[j // page].long(), j % page] = torch.randn(n, Hk, D, generator=g)
        for b, n in enumerate(kv_lens):
            fill(self.pages[b], n)
            self.pages[b, -(-n // page):] = -7          # never looked at
        fill(self.pp, prefix)
        self.k, self.v = k.to(dtype), v.to(dtype)
        self.q = torch.randn(sum(self.q_lens), Hq, D, generator=g).to(dtype)
        self.heads_first = heads_first
        self.max_q, self.max_kv = max(self.q_lens), max(kv_lens)
        if runs:                            # by a bound, and a table for as many keys
            assert B > 1 and 16 < self.max_q * Hq // Hk <= 128 and not prefix
            self.max_kv = 128 * max(32, -(-4096 // (B * Hk)))
            more = self.max_kv // page - wide
            self.pages = torch.cat((self.pages, torch.full((B, more), -7, dtype=torch.int32)), 1)
        self.seen = seen_of(trees, self.max_q)

    def place(self, x):
        if self.heads_first:
            return x.transpose(1, 2).contiguous().cuda().transpose(1, 2)
        return x.cuda()

    def run(self, seen=None, **kw):
        from warp_b200 import ops
        out = ops.tree_attention(
            self.q.cuda(), self.place(self.k), self.place(self.v), self.pages.cuda(),
            i32(self.kv_lens).cuda(), i32(starts_of(self.q_lens)).cuda(),
            (self.seen if seen is None else seen).cuda(), self.max_q, self.max_kv,
            prefix_pages=self.pp.cuda() if self.prefix else None, prefix_len=self.prefix, **kw)
        ops.attn_status()
        return out.cpu()

    def keys(self, b, i, seen):
        """Own keys that node i of request b sees."""
        n, L = self.q_lens[b], self.kv_lens[b]
        row = seen[starts_of(self.q_lens)[b] + i]
        nodes = [m for m in range(n) if int(row[m // 64]) >> (m % 64) & 1]
        return list(range(max(0, L - n))) + [L - n + m for m in nodes if L - n + m >= 0]

    def want(self, seen=None):
        seen = self.seen if seen is None else seen
        q, D = self.q.double(), self.q.shape[2]
        G = q.shape[1] // self.k.shape[2]
        o, mag = torch.zeros_like(q), torch.zeros_like(q)

        def rows(x, table, j):
            j = torch.tensor(j, dtype=torch.long)
            return x[table[j // self.page].long(), j % self.page].double()
        t = 0
        for b, n in enumerate(self.q_lens):
            for i in range(n):
                j = self.keys(b, i, seen)
                k, v = (torch.cat((rows(x, self.pp, list(range(self.prefix))),
                                   rows(x, self.pages[b], j))).repeat_interleave(G, 1)
                        for x in (self.k, self.v))
                if len(k):
                    p = (torch.einsum("hd,jhd->hj", q[t], k) / math.sqrt(D)).softmax(-1)
                    o[t] = torch.einsum("hj,jhd->hd", p, v)
                    mag[t] = torch.einsum("hj,jhd->hd", p, v.abs())
                t += 1
        return o, mag

    def check(self, seen=None, **kw):
        got = self.run(seen, **kw)
        o, mag = self.want(seen)
        u = torch.finfo(got.dtype).eps / 2
        bad = ~((got.double() - o).abs() <= u * o.abs() + (u + 2.0 ** -12) * mag)
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3],
                               (got.double() - o).abs().max().item())
        return got


def trees_of(sizes, kind="any", seed=0):
    rng = random.Random(seed)
    return [random_parents(rng, n, kind) if n else [] for n in sizes]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sizes, kv", [
    ([1], [1]), ([1, 2, 3], [5, 40, 3]), ([4, 0, 2], [300, 9, 16]), ([8], [8]), ([13, 1], [29, 400]),
    ([64, 63], [64, 700]), ([65], [193]), ([26, 3, 90], [777, 17, 90]), ([130], [131])])
def test_trees(cuda, dtype, D, sizes, kv):
    Trees(trees_of(sizes), kv, 6, 2, D, 16, dtype, seed=sum(kv)).check()


@pytest.mark.parametrize("kind", ["chain", "star", "forest"])
@pytest.mark.parametrize("sizes, kv", [([2, 5], [33, 70]), ([40, 7], [90, 7]), ([150], [1000])])
def test_tree_shapes(cuda, kind, sizes, kv):
    Trees(trees_of(sizes, kind), kv, 8, 2, 128, 32, torch.bfloat16, seed=3).check()


@pytest.mark.parametrize("Hq, Hk", [(1, 1), (4, 4), (18, 2), (56, 8), (16, 1), (40, 1), (130, 1)])
def test_tree_heads(cuda, Hq, Hk):
    Trees(trees_of([2, 7, 21]), [77, 7, 150], Hq, Hk, 64, 16, torch.float16, seed=Hq).check()


@pytest.mark.parametrize("page, heads_first", [(16, True), (32, False), (64, True), (128, False),
                                               (1024, False), (4096, True)])
def test_tree_pages(cuda, page, heads_first):
    """Trees that begin and end inside a page, on both sides of a page's end."""
    sizes = [1, 20, 33, 5]
    kv = [page, page + 7, 2 * page + 16 if page < 1024 else 300, page + 5]
    Trees(trees_of(sizes), kv, 8, 2, 128, page, torch.bfloat16, heads_first, seed=page).check()


@pytest.mark.parametrize("sizes, kv, prefix", [
    ([5], [7], 300),                        # one request: the prefix in its own pass
    ([3, 2, 5], [3, 2, 9], 70), ([1, 6, 4, 2], [40, 6, 5, 300], 515),
    ([100, 90], [100, 95], 130), ([1, 200, 1], [5, 300, 2], 64)])
def test_tree_behind_a_prefix(cuda, sizes, kv, prefix):
    Trees(trees_of(sizes), kv, 18, 2, 64, 16, torch.bfloat16, prefix=prefix, seed=prefix).check()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [3, 40])
def test_tree_behind_long_context(cuda, D, n):
    """Parts of the keys' range, the tree in the last one."""
    Trees(trees_of([n, n]), [20001, 4096 + n // 2], 8, 2, D, 64, torch.bfloat16, seed=n).check()


# Batches whose keys the card's blocks take equal runs of: items that begin and end within
# a run, runs within an item, requests without nodes or keys in between.
RAGGED = [1500, 3, 0, 129, 700, 128, 40, 1, 1023]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("nodes, Hq, Hk", [(8, 24, 4), (32, 16, 4), (21, 24, 4), (100, 8, 8)])
def test_runs(cuda, dtype, D, nodes, Hq, Hk):
    sizes = [max(0, min(nodes - 3 * (b % 4), k)) for b, k in enumerate(RAGGED)]
    sizes[4] = 0
    Trees(trees_of(sizes), RAGGED, Hq, Hk, D, 16, dtype, seed=nodes, runs=True).check()


@pytest.mark.parametrize("batch", [31, 33, 70])
def test_runs_of_many_requests(cuda, batch):
    """More requests than a warp has lanes; most items lie within one run."""
    rng = random.Random(batch)
    kv = [rng.choice([0, 20, 127, 128, 129, 300]) for _ in range(batch)]
    sizes = [min(k, rng.randint(0, 9)) for k in kv]
    sizes[0], kv[0] = 9, 300
    Trees(trees_of(sizes), kv, 16, 4, 64, 32, torch.bfloat16, seed=batch, runs=True).check()


@pytest.mark.parametrize("sizes, kv", [([30, 0], [20011, 0]), ([0, 30], [50, 5000]),
                                       ([9, 9], [40000, 1]), ([5, 9, 0], [0, 0, 0]),
                                       ([30, 1], [100, 0])])
def test_runs_of_few_items(cuda, sizes, kv):
    """Every block has a part of the same items, or none has any."""
    Trees(trees_of(sizes), kv, 8, 2, 128, 64, torch.bfloat16, seed=kv[0], runs=True).check()


@pytest.mark.parametrize("nodes", [9, 30])
def test_runs_are_the_same_every_time(cuda, nodes):
    sizes = [min(nodes, k) for k in RAGGED]
    c = Trees(trees_of(sizes), RAGGED, 16, 4, 128, 16, torch.bfloat16, seed=7, runs=True)
    want = c.run()
    for _ in range(5):
        assert torch.equal(c.run(), want)


def test_runs_with_more_nodes_than_keys_and_empty_masks(cuda):
    sizes = [30, 20, 7, 30, 30, 12]
    c = Trees(trees_of(sizes, "chain"), [1000, 9, 0, 15, 700, 1], 16, 4, 128, 16, torch.float16,
              seed=3, runs=True)
    seen = c.seen.clone()
    seen[80:90] = 0                         # of the fourth request, without a key before them
    got = c.check(seen)
    first = starts_of(sizes)
    assert not got[first[2]:first[3]].any() and not got[first[1]:first[1] + 11].any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("short", [1, 60, 129])
def test_runs_with_short_requests_between_long_ones(cuda, D, short):
    """Several tasks a block: a short one's tile of keys, partly filled, is waited for while
    the long one before it still goes through the ring."""
    kv = [n for i in range(14) for n in (2600 - 90 * i, short + i // 4)]
    sizes = [min(5, n) for n in kv]
    c = Trees(trees_of(sizes), kv, 16, 4, D, 16, torch.bfloat16, seed=short, runs=True)
    want = c.check()
    for _ in range(20):
        assert torch.equal(c.run(), want)


def test_runs_of_many_short_requests(cuda):
    """Tasks of one tile behind one another, and items that two blocks share: the same bits."""
    kv = [(18, 20, 1017, 61, 17, 1, 2158, 243, 14, 1, 102, 2686, 68, 371, 210)[i % 15] + i // 15
          for i in range(90)]
    sizes = [min(3 + i * 7 % 16, n) for i, n in enumerate(kv)]
    c = Trees(trees_of(sizes), kv, 56, 8, 64, 256, torch.bfloat16, seed=7, runs=True)
    want = c.check()
    for _ in range(20):
        assert torch.equal(c.run(), want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_runs_keep_what_is_not_seen_apart(cuda, dtype, bad):
    """Values that are not finite, in several requests at once, reach who sees them alone."""
    sizes = [20, 31, 9, 30, 25, 1]
    c = Trees(trees_of(sizes, seed=5), [900, 300, 9, 158, 700, 1], 16, 4, 64, 16, dtype, seed=5,
              runs=True)
    clean, first = c.run(), starts_of(sizes)
    sees = torch.zeros(sum(sizes), dtype=torch.bool)
    for b, m in ((0, 7), (1, 30), (3, 12), (4, 3)):
        j = c.kv_lens[b] - sizes[b] + m
        c.v[c.pages[b, j // 16].long(), j % 16][2, 5] = bad
        for i in range(sizes[b]):
            sees[first[b] + i] = bool(int(c.seen[first[b] + i, 0]) >> m & 1)
    got = c.run()
    assert torch.equal(got[~sees], clean[~sees])
    mine = torch.zeros(16, dtype=torch.bool)
    mine[8:12] = True                       # of kv head 2
    assert torch.equal(got[sees][:, ~mine], clean[sees][:, ~mine])
    hit = got[sees][:, mine][..., 5].float()
    assert (hit.isnan() if math.isnan(bad) else hit == bad).all()


def test_runs_replay_while_lengths_change(cuda):
    """A captured call reads the lengths, the nodes and the masks of its replay."""
    from warp_b200 import ops
    sizes = [min(9, k) for k in RAGGED]
    c = Trees(trees_of(sizes), RAGGED, 16, 4, 128, 16, torch.bfloat16, seed=9, runs=True)
    args = [c.q.cuda(), c.k.cuda(), c.v.cuda(), c.pages.cuda(), i32(c.kv_lens).cuda(),
            i32(starts_of(sizes)).cuda(), c.seen.cuda()]
    out = torch.zeros_like(args[0])

    def call():
        ops.tree_attention(*args, 9, c.max_kv, out=out)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for shorter in (0, 5, 300, 1499):
        kv = [max(n, k - shorter) for n, k in zip(sizes, RAGGED)]
        args[4].copy_(i32(kv))
        c.kv_lens = kv
        out.fill_(7.0)
        graph.replay()
        c.run = lambda seen: out.cpu()
        c.check()
    ops.attn_status()


@pytest.mark.parametrize("sizes, kv", [([5], [2]), ([40, 3], [33, 1]), ([200], [100]), ([2, 1], [0, 4])])
def test_more_nodes_than_keys(cuda, sizes, kv):
    """Nodes whose key would lie before the first have none."""
    Trees(trees_of(sizes, "chain"), kv, 8, 2, 128, 16, torch.bfloat16, seed=11).check()


@pytest.mark.parametrize("sizes", [[3, 2], [40, 30]])
def test_masks_that_leave_nothing(cuda, sizes):
    """Rows without a bit: zeros where there is no key before the tree."""
    c = Trees(trees_of(sizes), [sizes[0], sizes[1] + 9], 4, 2, 64, 16, torch.float16, seed=2)
    seen = c.seen.clone()
    seen[1] = 0
    seen[sizes[0] + 1] = 0
    got = c.check(seen)
    assert not got[1].any() and got[sizes[0] + 1].any()


@pytest.mark.parametrize("sizes", [[2, 3], [70, 66]])
def test_bits_past_the_nodes_mean_nothing(cuda, sizes):
    c = Trees(trees_of(sizes), [sizes[0] + 5, sizes[1]], 4, 2, 64, 16, torch.float16, seed=4)
    seen = torch.cat((c.seen, torch.full_like(c.seen, -1)), 1)
    t = 0
    for n in sizes:
        for i in range(n):
            if n % 64:
                seen[t, n // 64] |= -1 << n % 64
            t += 1
    assert torch.equal(c.run(seen), c.run())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n, group", [(4, 2), (30, 4), (140, 2)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_a_node_does_not_see_has_no_effect(cuda, dtype, n, group, bad):
    """A node's key and value that are not finite reach the nodes that see it, no other."""
    c = Trees(trees_of([n, 3], seed=n), [n + 21, 3], 2 * group, 2, 64, 16, dtype, seed=n)
    clean = c.run()
    m = n // 2
    j = c.kv_lens[0] - n + m
    at = c.pages[0, j // 16].long(), j % 16
    sees = torch.tensor([int(c.seen[i, m // 64]) >> (m % 64) & 1 for i in range(n)] + [0] * 3).bool()
    assert sees.any() and not sees.all()
    for x in (c.v, c.k):
        kept = x[at].clone()
        x[at][0, 5] = bad
        got = c.run()
        assert torch.equal(got[~sees], clean[~sees])
        if x is c.v:
            hit = got[sees][:, :group, 5].float()       # of kv head 0
            assert (hit.isnan() if math.isnan(bad) else hit == bad).all()
            assert torch.equal(got[sees][:, group:], clean[sees][:, group:])
        x[at] = kept


@pytest.mark.parametrize("sizes, kv", [([3, 5], [50, 5]), ([90, 40], [300, 40])])
def test_a_chain_is_causal(cuda, sizes, kv):
    """Attention of the same rows without a tree is as near to the tree's definition."""
    from warp_b200 import ops
    c = Trees(trees_of(sizes, "chain"), kv, 8, 2, 128, 16, torch.bfloat16, seed=8)
    c.check()
    c.run = lambda seen: ops.paged_attention(
        c.q.cuda(), c.k.cuda(), c.v.cuda(), c.pages.cuda(), i32(kv).cuda(),
        i32(starts_of(sizes)).cuda(), c.max_q, max(kv)).cpu()
    c.check()


def test_tree_rows_of_no_request_and_bounds(cuda):
    from warp_b200 import ffi, ops
    c = Trees(trees_of([6, 4]), [30, 20], 4, 2, 64, 16, torch.float16, seed=6)
    good = c.run()
    args = (c.q.cuda(), c.k.cuda(), c.v.cuda(), c.pages.cuda(), i32(c.kv_lens).cuda())
    out = torch.full_like(c.q, 9.0).cuda()
    ops.tree_attention(*args, i32([0, 6, 6]).cuda(), c.seen.cuda(), 6, 30, out=out)
    ops.attn_status()
    assert torch.equal(out[:6].cpu(), good[:6]) and (out[6:] == 9).all()
    ops.tree_attention(*args, i32([0, 6, 10]).cuda(), c.seen.cuda(), 5, 30)
    with pytest.raises(ffi.WarpError, match="length"):
        ops.attn_status()


# ---- pick ------------------------------------------------------------------------------


class Logits:
    def __init__(self, sizes, V, dtype, seed=0, history=50, penalties=True, bias=None,
                 masked=False, tree=True, far=False, large=False):
        rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
        self.sizes, self.V = sizes, V
        B, T = len(sizes), sum(sizes)
        self.x = (3 * torch.randn(T, V, generator=g)).to(dtype)
        self.kw = dict(q_start=i32(starts_of(sizes)), max_q=max(sizes))
        top = V + 3 if far else V - 1       # tokens outside the vocabulary count for nothing
        self.history = [[rng.choice([0, V - 1, rng.randint(-2 if far else 0, top)])
                         for _ in range(rng.randint(0, history))] for _ in range(B)]
        self.drafted = [rng.choice([0, V - 1, rng.randint(-2 if far else 0, top)]) for _ in range(T)]
        self.trees = [random_parents(rng, n, "any") if n else [] for n in sizes]
        if penalties:
            # a history with more places than this goes the way of large calls
            wide = 16400 if large else max(1, max(map(len, self.history)))
            self.kw.update(history=i32([h + [0] * (wide - len(h)) for h in self.history]),
                           history_len=i32([len(h) for h in self.history]),
                           repetition=1 + torch.rand(B, generator=g),
                           frequency=torch.randn(B, generator=g), presence=torch.rand(B, generator=g))
        else:
            self.history = [[] for _ in sizes]
        self.tree = tree
        if tree:
            self.kw.update(drafted=i32(self.drafted), seen=seen_of(self.trees, max(sizes)))
        if bias:
            self.kw["bias"] = torch.randn((B, V) if bias == "each" else (V,), generator=g)
        if masked:
            self.kw["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (T, -(-V // 32)), generator=g).int()

    def want(self):
        """The same fp32 operations, one by one."""
        rows, t, f = [], 0, np.float32
        for b, n in enumerate(self.sizes):
            for i, path in enumerate(paths_of(self.trees[b])):
                x = self.x[t].float().numpy().copy()
                context = list(self.history[b])
                if self.tree:
                    context += [self.drafted[t - i + m] for m in path]
                count = np.bincount([v for v in context if 0 <= v < self.V], minlength=self.V)
                hit = count > 0
                rep, freq, pres = (f(self.kw[k][b].item()) if k in self.kw else f(d) for k, d in
                                   (("repetition", 1), ("frequency", 0), ("presence", 0)))
                y = x[hit]
                y = np.where(y > 0, y / rep, y * rep) - freq * count[hit].astype(f)
                x[hit] = y - pres
                if "bias" in self.kw:
                    w = self.kw["bias"]
                    x = x + (w[b] if w.dim() == 2 else w).numpy()
                if "allowed" in self.kw:
                    words = self.kw["allowed"][t].numpy().view(np.uint32)
                    v = np.arange(self.V)
                    x[(words[v // 32] >> (v % 32).astype(np.uint32)) & 1 == 0] = -np.inf
                rows.append(torch.from_numpy(x))
                t += 1
        return torch.stack(rows)

    def check(self, keep=True, place=lambda x: x.cuda(), in_place=False):
        from warp_b200 import ops
        x = place(self.x)
        out = (x if in_place else place(torch.zeros_like(self.x))) if keep else None
        kw = {k: v.cuda() if torch.is_tensor(v) else v for k, v in self.kw.items()}
        picked = ops.pick_tokens(x, out=out, **kw)
        ops.attn_status()
        want = self.want()
        if keep:
            assert torch.equal(out.cpu(), want.to(self.x.dtype))
        else:
            assert torch.equal(x.cpu(), self.x)
        first = [-1 if r.max() == -math.inf else int((r == r.max()).nonzero()[0]) for r in want]
        assert picked.tolist() == first
        return picked


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 31, 100, 1000, 4099, 50001])
@pytest.mark.parametrize("keep", [False, True])
def test_pick(cuda, dtype, V, keep):
    Logits([1, 5, 0, 3], V, dtype, seed=V, bias="each", masked=V > 2).check(keep)


@pytest.mark.parametrize("kw", [
    dict(penalties=False, tree=False), dict(penalties=False), dict(tree=False),
    dict(bias="all"), dict(masked=True), dict(far=True), dict(history=5000),
    dict(penalties=False, tree=False, bias="each", masked=True)])
@pytest.mark.parametrize("sizes", [[1], [1] * 7, [70], [26, 3, 19, 1]])
def test_pick_parts(cuda, kw, sizes):
    Logits(sizes, 3001, torch.float32, seed=5, **kw).check()


def test_pick_large_vocabulary(cuda):
    """More than the blocks of a cluster count at a time."""
    Logits([2, 1], 300001, torch.bfloat16, seed=1, bias="all", masked=True, history=2000).check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset, row", [(0, 1003), (1, 1003), (3, 1024), (5, 1001), (8, 1008)])
@pytest.mark.parametrize("in_place", [False, True])
def test_pick_strides(cuda, dtype, offset, row, in_place):
    """Rows at any element, with something between them that stays."""
    base = []

    def place(x):
        room = torch.full((len(x) * row + 40,), 77.0, dtype=dtype, device="cuda")
        y = torch.as_strided(room, x.shape, (row, 1), offset)
        y.copy_(x)
        base.append((room, y))
        return y
    Logits([3, 4], 1000, dtype, seed=offset, bias="all").check(place=place, in_place=in_place)
    for room, y in base:
        y.fill_(77.0)
        assert (room == 77).all()


# Calls that go the way of large ones: by a history of many places, or by a vocabulary.
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sizes, V", [([3, 0, 40, 1, 26], 16001), ([12], 100003), ([1] * 33, 32000),
                                      ([2, 3], 262149), ([1] * 600, 2049)])
@pytest.mark.parametrize("keep", [False, True])
def test_pick_many(cuda, dtype, sizes, V, keep):
    Logits(sizes, V, dtype, seed=V, bias="each", masked=True, history=3000, large=True).check(keep)


@pytest.mark.parametrize("kw", [
    dict(penalties=False, tree=False), dict(penalties=False), dict(tree=False), dict(),
    dict(bias="all"), dict(masked=True), dict(far=True), dict(history=16000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pick_many_parts(cuda, dtype, kw):
    Logits([5, 1, 3], 131204, dtype, seed=6, large=True, **kw).check()


def test_pick_long_histories(cuda):
    """Tokens that occur more often than 16 bits count, in a history that says so."""
    from warp_b200 import ops
    V, rep = 40000, torch.full((30,), 2.0, device="cuda")
    x = torch.zeros(30, V, device="cuda")
    x[:, 77], x[:, 5] = 9.0, 8.0
    history = torch.full((30, 70001), 77, dtype=torch.int32, device="cuda")
    history[:, ::3] = torch.arange(23334, device="cuda").int()
    freq = torch.full((30,), 2.0 ** -14, device="cuda")
    out = torch.empty_like(x)
    lens = i32([70001 - 7 * b for b in range(30)]).cuda()
    picked = ops.pick_tokens(x, history=history, history_len=lens, repetition=rep, frequency=freq,
                             out=out)
    ops.attn_status()
    count = torch.stack([torch.bincount(h[:n].long(), minlength=V) for h, n in zip(history, lens)])
    want = torch.where(count > 0, x / 2 - freq[:, None] * count.float(), x)
    assert torch.equal(out, want) and count[:, 77].min() > 46000
    assert picked.tolist() == want.argmax(1).tolist()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset, row", [(0, 2003), (1, 2003), (3, 2048), (5, 2001), (8, 2008)])
@pytest.mark.parametrize("in_place", [False, True])
def test_pick_many_strides(cuda, dtype, offset, row, in_place):
    base = []

    def place(x):
        room = torch.full((len(x) * row + 40,), 77.0, dtype=dtype, device="cuda")
        y = torch.as_strided(room, x.shape, (row, 1), offset)
        y.copy_(x)
        base.append((room, y))
        return y
    Logits([30, 1, 29], 2000, dtype, seed=offset, bias="all", large=True).check(
        place=place, in_place=in_place)
    for room, y in base:
        y.fill_(77.0)
        assert (room == 77).all()


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e30, 3e38])
@pytest.mark.parametrize("repetition", [1.0, 1.1, 3.0, 1e-7, 1e7, 1e30])
def test_pick_divides_as_a_division(cuda, scale, repetition):
    """At the numbers' ends, where a product by the reciprocal would be off."""
    from warp_b200 import ops
    g = torch.Generator().manual_seed(4)
    x = (torch.randn(40, 30000, generator=g) * scale).cuda()    # by the places of the history
    rep = torch.full((40,), repetition, device="cuda")
    history = torch.arange(30000, dtype=torch.int32, device="cuda").expand(40, 30000).contiguous()
    out = torch.empty_like(x)
    ops.pick_tokens(x, history=history, repetition=rep, out=out,
                    history_len=torch.full((40,), 30000, dtype=torch.int32, device="cuda"))
    ops.attn_status()
    assert torch.equal(out, torch.where(x > 0, x / rep[:, None], x * rep[:, None]))


def test_pick_reciprocals_divide_exactly(cuda):
    """The corrected product by a reciprocal against the division, over many divisors."""
    from warp_b200 import ops
    g = torch.Generator().manual_seed(8)
    B, V = 4096, 4096
    rep = (1 + torch.rand(B, generator=g)).cuda()
    rep[:1024] = torch.exp2(torch.rand(1024, generator=g) * 40 - 20).cuda()
    rep[0], rep[1], rep[2] = 1.0, 2 - 2.0 ** -23, 1 + 2.0 ** -23
    x = (torch.randn(B, V, generator=g) * 8).abs().cuda()
    history = torch.arange(V, dtype=torch.int32, device="cuda").expand(B, V).contiguous()
    out = torch.empty_like(x)
    ops.pick_tokens(x, history=history, repetition=rep, out=out,
                    history_len=torch.full((B,), V, dtype=torch.int32, device="cuda"))
    assert torch.equal(out, x / rep[:, None])


def test_pick_many_ties_and_what_is_not_finite(cuda):
    from warp_b200 import ops
    x = torch.zeros(1300, 5000)
    x[1, 4000] = x[1, 17] = x[1, 4999] = 2.0
    x[2] = -math.inf
    x[3] = -math.inf
    x[3, 4321] = -1e30
    x[4] = math.nan
    x[5, ::2] = math.nan
    x[6] = -0.0
    x[6, 3000] = 0.0
    x[7, 2500:] = math.inf
    want = [0, 17, -1, 4321, -1, 1, 0, 2500] + [0] * 1292
    assert ops.pick_tokens(x.cuda()).tolist() == want
    none = torch.zeros(157, dtype=torch.int32, device="cuda")
    assert ops.pick_tokens(x.cuda(), allowed=none).tolist() == [-1] * 1300


def test_pick_without_requests(cuda):
    """A row a request, and no context: the plain largest."""
    from warp_b200 import ops
    x = torch.randn(9, 777, generator=torch.Generator().manual_seed(0)).cuda()
    assert ops.pick_tokens(x).tolist() == x.argmax(1).tolist()
    assert ops.pick_tokens(x[:0]).shape == (0,)


def test_pick_ties_and_what_is_not_finite(cuda):
    from warp_b200 import ops
    x = torch.zeros(8, 5000)
    x[1, 4000] = x[1, 17] = x[1, 4999] = 2.0
    x[2] = -math.inf
    x[3] = -math.inf
    x[3, 4321] = -1e30
    x[4] = math.nan
    x[5, ::2] = math.nan
    x[6] = -0.0
    x[6, 3000] = 0.0
    x[7, 2500:] = math.inf
    assert ops.pick_tokens(x.cuda()).tolist() == [0, 17, -1, 4321, -1, 1, 0, 2500]
    none = torch.zeros(157, dtype=torch.int32, device="cuda")
    out = torch.empty(8, 5000, device="cuda")
    assert ops.pick_tokens(x.cuda(), allowed=none, out=out).tolist() == [-1] * 8
    assert (out == -math.inf).all()


def test_pick_leaves_rows_of_no_request(cuda):
    from warp_b200 import ffi, ops
    x = torch.randn(6, 300, generator=torch.Generator().manual_seed(1)).cuda()
    out = torch.full_like(x, 5.0)
    picked = ops.pick_tokens(x, i32([1, 3, 4]).cuda(), max_q=2, out=out)
    ops.attn_status()
    assert picked[1:4].tolist() == x[1:4].argmax(1).tolist()
    assert torch.equal(out[1:4], x[1:4]) and (out[0] == 5).all() and (out[4:] == 5).all()
    ops.pick_tokens(x, i32([0, 6]).cuda(), max_q=2)
    with pytest.raises(ffi.WarpError, match="length"):
        ops.attn_status()
    ops.pick_tokens(x[:1], history=i32([[1, 2]]).cuda(), history_len=i32([3]).cuda())
    with pytest.raises(ffi.WarpError, match="length"):
        ops.attn_status()


# ---- accept ------------------------------------------------------------------------------


class Drafted:
    """Trees with few different tokens, so that paths of all lengths are accepted."""

    def __init__(self, sizes, extra, layers=2, Hk=2, D=64, page=16, dtype=torch.float16,
                 heads_first=False, tokens=3, kind="any", seed=0):
        rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
        self.sizes, self.page = sizes, page
        self.trees = [random_parents(rng, n, kind) if n else [] for n in sizes]
        self.kv = [n + rng.randint(0, extra) for n in sizes]
        T, B, wide = sum(sizes), len(sizes), max(1, -(-max(self.kv) // page))
        self.drafted = [rng.randrange(-1, tokens) for _ in range(T)]
        self.picked = [rng.randrange(-1, tokens) for _ in range(T)]
        self.max_q = max(1, max(sizes))
        self.seen = seen_of(self.trees, self.max_q)
        n = B * wide + 1
        self.pages = torch.randperm(n, generator=g).int()[:B * wide].view(B, wide)
        shape = (layers, 2, n, Hk, page, D) if heads_first else (layers, 2, n, page, Hk, D)
        self.pools = torch.randn(shape, generator=g).to(dtype).cuda()
        if heads_first:
            self.pools = self.pools.transpose(3, 4)

    def want(self):
        """The longest path, found from the root on, and the caches after it."""
        pools = self.pools.cpu().clone()
        count, path, chosen, after = [], [], [], []
        t0 = 0
        for b, n in enumerate(self.sizes):
            best, reached = [], {}
            for i in range(n):
                p = self.trees[b][i]
                token = self.drafted[t0 + i]
                if i == 0:
                    reached[0] = [0]
                elif p in reached and token >= 0 and token == self.picked[t0 + p]:
                    reached[i] = reached[p] + [i]
                if len(reached.get(i, ())) > len(best):
                    best = reached[i]
            base = self.kv[b] - n
            for d, i in enumerate(best):
                (pa, sa), (pb, sb) = (divmod(base + x, self.page) for x in (i, d))
                pools[:, :, self.pages[b, pb].item(), sb] = pools[:, :, self.pages[b, pa].item(),
                                                                  sa].clone()
            rest = [-1] * (self.max_q - len(best))
            count.append(len(best))
            path.append(best + rest)
            chosen.append([self.picked[t0 + i] for i in best] + rest)
            after.append(base + len(best))
            t0 += n
        return count, path, chosen, after, pools

    def check(self, as_list=False):
        from warp_b200 import ops
        *want, pools = self.want()
        caches = self.pools[:, 0], self.pools[:, 1]
        if as_list:
            caches = [(c[0].clone(), c[1].clone()) for c in self.pools]
        got = ops.tree_accept(i32(self.drafted).cuda(), i32(self.picked).cuda(), self.seen.cuda(),
                              i32(starts_of(self.sizes)).cuda(), i32(self.kv).cuda(), self.max_q,
                              caches=caches, pages=self.pages.cuda())
        ops.attn_status()
        assert [x.tolist() for x in got] == want
        if as_list:
            for (k, v), w in zip(caches, pools):
                assert torch.equal(k.cpu(), w[0]) and torch.equal(v.cpu(), w[1])
        else:
            assert torch.equal(self.pools.cpu(), pools)
        return want


@pytest.mark.parametrize("sizes", [[1], [2, 0, 1], [26], [64, 65, 3], [5] * 40, [300, 129]])
@pytest.mark.parametrize("tokens", [1, 2, 3])
def test_accept(cuda, sizes, tokens):
    Drafted(sizes, 50, tokens=tokens, seed=len(sizes)).check()


@pytest.mark.parametrize("kind", ["any", "star", "forest"])
@pytest.mark.parametrize("sizes", [[26], [64, 65, 3], [300, 129]])
def test_accept_the_deepest(cuda, kind, sizes):
    """Every token agrees: the deepest path from node 0, the first of equals."""
    c = Drafted(sizes, 50, kind=kind, seed=9)
    c.drafted, c.picked = [4] * sum(sizes), [4] * sum(sizes)
    want = c.check()
    assert want[0] == [max(len(p) for p in paths_of(t) if p[0] == 0) for t in c.trees]


def test_accept_a_whole_chain(cuda):
    """Nothing moves, and moves by one: node 1 is refused, the rest is accepted."""
    c = Drafted([9, 9], 20, kind="chain", tokens=1, seed=3)
    c.drafted, c.picked = [0] * 18, [0] * 18
    c.trees[1][2] = 0                       # node 1 is a sibling of the others' first
    c.drafted[9 + 1] = 1
    c.seen = seen_of(c.trees, 9)
    want = c.check()
    assert want[0] == [9, 8] and want[1][1] == [0, 2, 3, 4, 5, 6, 7, 8, -1]


@pytest.mark.parametrize("kw", [
    dict(D=128, Hk=8, page=32), dict(D=10, Hk=3), dict(D=64, heads_first=True),
    dict(D=256, Hk=1, dtype=torch.bfloat16, page=64), dict(layers=1), dict(layers=131, Hk=1),
    dict(D=2, Hk=1)])
@pytest.mark.parametrize("as_list", [False, True])
def test_accept_layouts(cuda, kw, as_list):
    if kw.get("D") in (10, 2):              # strides are multiples of 16 bytes: rows with a margin
        c = Drafted([20, 3, 41], 30, tokens=2, seed=7, **kw)
        room = torch.zeros(c.pools.shape[:-1] + (16,), dtype=c.pools.dtype, device="cuda")
        room[..., :c.pools.shape[-1]] = c.pools
        c.pools = room[..., :c.pools.shape[-1]]
        if as_list:                         # a clone would lose the margin
            return
        c.check()
        assert not room[..., c.pools.shape[-1]:].any()
        return
    Drafted([20, 3, 41], 30, tokens=2, seed=7, **kw).check(as_list)


def test_accept_without_caches(cuda):
    from warp_b200 import ops
    c = Drafted([30, 4], 10, tokens=2, seed=1)
    got = ops.tree_accept(i32(c.drafted).cuda(), i32(c.picked).cuda(), c.seen.cuda(),
                          i32([0, 30, 34]).cuda(), i32(c.kv).cuda(), 30)
    assert [x.tolist() for x in got] == list(c.want()[:4])


def test_accept_with_bad_pages(cuda):
    from warp_b200 import ffi, ops
    ops.attn_status()
    c = Drafted([3], 0, tokens=1, seed=1)
    c.drafted, c.picked = [0, -1, 0], [0, 0, 0]
    c.seen = seen_of([[-1, 0, 0]], 3)
    before = c.pools.clone()
    for pages, text in (([[99]], "page number"), ([[-1]], "page number")):
        got = ops.tree_accept(i32(c.drafted).cuda(), i32(c.picked).cuda(), c.seen.cuda(),
                              i32([0, 3]).cuda(), i32([3]).cuda(), 3,
                              caches=(c.pools[:, 0], c.pools[:, 1]), pages=i32(pages).cuda())
        assert got[1].tolist() == [[0, 2, -1]]
        with pytest.raises(ffi.WarpError, match=text):
            ops.attn_status()
    # keys past the row's pages, and more nodes than keys
    for kv in (19, 2):
        ops.tree_accept(i32(c.drafted).cuda(), i32(c.picked).cuda(), c.seen.cuda(),
                        i32([0, 3]).cuda(), i32([kv]).cuda(), 3,
                        caches=(c.pools[:, 0], c.pools[:, 1]), pages=i32([[0]]).cuda())
        with pytest.raises(ffi.WarpError, match="length"):
            ops.attn_status()
    moved = (c.pools != before).flatten(4).any(-1).nonzero()[:, 2:].unique(dim=0).tolist()
    assert moved in ([], [[0, 0]])          # kv 2: node 2's key 1 to place 0
