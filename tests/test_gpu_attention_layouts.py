"""Attention of many rows over every layout that the pages and queries may have.

Requests of more than 16 rows a kv head, and prefixes of a batch with as many, are
the tensor-core kernel's.  Tolerances are those of the attention tests."""
import math

import pytest
import torch

from test_gpu_attention import Case, gen

pytestmark = pytest.mark.gpu

PAGES = [(16, True), (32, False), (64, True), (128, False), (256, True), (1024, False), (4096, True)]


@pytest.mark.parametrize("page, heads_first", PAGES)
@pytest.mark.parametrize("D", [64, 128])
def test_pages(cuda, page, heads_first, D):
    """Boxes that are a page, and boxes inside one."""
    kv = [300, 77, 1500 if page < 1024 else page + 129]
    Case([90, 40, 33], kv, 8, 2, D, page, torch.bfloat16, heads_first, seed=page).check()


@pytest.mark.parametrize("page, heads_first", PAGES)
def test_pages_behind_a_prefix(cuda, page, heads_first):
    """One token a request, their rows together; and rows enough of their own."""
    Case([1] * 12, list(range(0, 60, 5)), 8, 2, 64, page, torch.float16, heads_first,
         prefix=391, seed=page).check()
    Case([70, 80], [99, 200], 8, 2, 128, page, torch.bfloat16, heads_first, prefix=391,
         seed=page).check(causal=False)


@pytest.mark.parametrize("D", [64, 128])
def test_strided_queries_and_given_out(cuda, D):
    """Heads of a projection's rows with others between, out of order in memory."""
    from warp_b200 import ops
    c = Case([60, 41], [60, 333], 8, 2, D, 32, torch.float16, seed=51)
    want = c.check()
    wide = torch.full((8, 101, 3, D + 16), math.nan, dtype=torch.float16)
    wide[:, :, 1, 8:D + 8] = c.q.transpose(0, 1)
    q = wide.cuda()[:, :, 1, 8:D + 8].transpose(0, 1)
    out = torch.empty(101, 8, D, dtype=torch.float16, device="cuda")
    got = ops.paged_attention(q, c.k.cuda(), c.v.cuda(), c.pages.cuda(), c.kv_len.cuda(),
                              c.q_start.cuda(), 60, 333, out=out)
    assert got is out and torch.equal(got.cpu(), want)
    ops.attn_status()


def test_pages_past_32_bits(cuda):
    """Pages whose offsets pass 2^31 elements, read by tiles."""
    from warp_b200 import ops
    page, Hk, D, n = 4096, 8, 128, 60
    total = 2 ** 31 // (page * Hk * D) + 8
    kp = torch.zeros(total, page, Hk, D, dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros_like(kp)
    pages = torch.tensor([[total - 1, 0, total - 2]], dtype=torch.int32, device="cuda")
    L = 2 * page + 100
    k = torch.randn(L, Hk, D, generator=gen(52)).bfloat16().cuda()
    v = torch.randn(L, Hk, D, generator=gen(53)).bfloat16().cuda()
    kv_len = torch.tensor([L], dtype=torch.int32, device="cuda")
    for i, p in enumerate(pages[0].tolist()):
        part = k[i * page:(i + 1) * page]
        kp[p, :len(part)], vp[p, :len(part)] = part, v[i * page:(i + 1) * page]
    q = torch.randn(n, Hk, D, generator=gen(54)).bfloat16().cuda()
    q_start = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    got = ops.paged_attention(q, kp, vp, pages, kv_len, q_start, n, L)
    sees = torch.arange(L, device="cuda") <= L - n + torch.arange(n, device="cuda")[:, None]
    s = torch.einsum("thd,jhd->htj", q.double(), k.double()) / math.sqrt(D)
    p = s.masked_fill(~sees, -math.inf).softmax(-1)
    o = torch.einsum("htj,jhd->thd", p, v.double())
    mag = torch.einsum("htj,jhd->thd", p, v.double().abs())
    tol = 2 * (2.0 ** -9 * o.abs() + (2.0 ** -9 + 2.0 ** -14) * mag)
    assert ((got.double() - o).abs() <= tol).all()
    ops.attn_status()


def test_captured_chunks(cuda):
    """A captured call of many rows and few; lengths move between replays."""
    from warp_b200 import ops
    c = Case([50, 1, 20], [400, 300, 120], 8, 2, 128, 32, torch.bfloat16, prefix=70, seed=55)
    x = [t.cuda() for t in (c.q, c.k, c.v, c.pages, c.kv_len, c.q_start)]
    front = c.pp.cuda()

    def call():
        return ops.paged_attention(*x, 50, 400, prefix_pages=front, prefix_len=70)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for lens in ([400, 300, 120], [50, 0, 20], [333, 1, 90], [60, 300, 3]):
        c.kv_lens = lens
        c.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        x[4].copy_(c.kv_len)
        graph.replay()
        torch.cuda.synchronize()
        o, mag = c.want()
        tol = 2 * (2.0 ** -9 * o.abs() + (2.0 ** -9 + 2.0 ** -14) * mag)
        assert ((out.double().cpu() - o).abs() <= tol).all(), lens
    ops.attn_status()
    del graph
