"""The attention operators against plain implementations in 64 bits.

Tolerances.  u is the result type's unit roundoff (2^-9 bf16, 2^-11 fp16).
Rotation: one rounding, u |y|, and a few fp32 operations on values no larger
than the row's largest, 2^-19 of it.  Attention: the weights are rounded to the
type before the second product, which moves a result by at most
u * sum p|v| / l, and the result is rounded once, u |o|; scores are fp32 sums
whose error of some 2^-15 in the exponent is the like of a further 2^-14 of
sum p|v| / l.  Both bounds are doubled for what was left out.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -9, torch.float32: 2.0 ** -24}


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- rotation and append -------------------------------------------------------------


def rope64(x, pos, f, w, eps, interleaved, scale):
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    if f is None:
        return x
    R = 2 * f.numel()
    a = pos.double()[:, None] * f
    c, s = (torch.cos(a) * scale)[:, None], (torch.sin(a) * scale)[:, None]
    i0, i1 = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2),
                                                                  slice(R // 2, R))
    y = x.clone()
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i0] * s + x[..., i1] * c
    return y


def rope_close(got, want):
    assert got.shape == want.shape
    tol = 2 * (ROUND[got.dtype] * want.abs() + 2.0 ** -19 * want.abs().amax(-1, keepdim=True))
    bad = (got.double().cpu() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3])


@pytest.mark.parametrize("types", [("float32", "float32"), ("float32", "float16"),
                                   ("float32", "bfloat16"), ("float16", "float16"),
                                   ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("D, R", [(64, 64), (128, 128), (128, 64), (128, 32), (128, 116), (80, 40),
                                  (256, 64), (256, 256), (96, 2), (10, 6), (2, 2), (64, None)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope(cuda, types, D, R, interleaved):
    from warp_b200 import ops
    ti, to = (getattr(torch, t) for t in types)
    g = gen(D + (R or 0))
    T, Hq, Hk = 7, 5, 2
    # parts of one projection's rows, with a margin behind them
    x = torch.randn(T, (Hq + Hk) * D + 16, generator=g).to(ti).cuda()
    q = x[:, :Hq * D].view(T, Hq, D)
    k = x[:, Hq * D:(Hq + Hk) * D].view(T, Hk, D)
    qn = (1 + 0.2 * torch.randn(D, generator=g)) if D != 96 else None
    kn = (1 + 0.2 * torch.randn(D, generator=g)) if D != 80 else None
    f, pos, scale = None, None, 1.0
    if R:
        f, scale = ops.rope_inv_freq(R, base=10000.0)
        scale = 1.25
        pos = torch.tensor([0, 1, 77, 4095, 131071, 2 ** 31 - 1, -5], dtype=torch.int32)
    qo, ko = ops.qk_norm_rope(q, k, pos.cuda() if R else None, f.cuda() if R else None,
                              q_norm=None if qn is None else qn.cuda(),
                              k_norm=None if kn is None else kn.cuda(), eps=1e-5,
                              interleaved=interleaved, rot_scale=scale, out_dtype=to)
    assert qo.dtype == to and qo.is_contiguous()
    rope_close(qo, rope64(q.cpu(), pos, f, qn, 1e-5, interleaved, scale))
    rope_close(ko, rope64(k.cpu(), pos, f, kn, 1e-5, interleaved, scale))


def test_rope_one_side_and_no_tokens(cuda):
    from warp_b200 import ops
    f, _ = ops.rope_inv_freq(64, device="cuda")
    q = torch.randn(3, 4, 64, generator=gen(1)).half().cuda()
    pos = torch.arange(3, dtype=torch.int32, device="cuda")
    qo, ko = ops.qk_norm_rope(q, None, pos, f)
    assert ko is None
    rope_close(qo, rope64(q.cpu(), pos.cpu(), f.cpu(), None, 0, False, 1.0))
    _, ko = ops.qk_norm_rope(None, q, pos, f)
    assert torch.equal(ko, qo)
    qo, ko = ops.qk_norm_rope(q[:0], q[:0], pos[:0], f)
    assert qo.shape == (0, 4, 64)


def test_rope_misaligned_rows(cuda):
    """An odd element offset: the widest vectors do not fit, the values do."""
    from warp_b200 import ops
    f, _ = ops.rope_inv_freq(64, device="cuda")
    x = torch.randn(5 * 131, generator=gen(2)).bfloat16().cuda()
    q = torch.as_strided(x, (5, 2, 64), (131, 65, 1), 1)
    pos = torch.arange(5, dtype=torch.int32, device="cuda") * 1000
    qo, _ = ops.qk_norm_rope(q, None, pos, f)
    rope_close(qo, rope64(q.cpu(), pos.cpu(), f.cpu(), None, 0, False, 1.0))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("tin", ["same", "float32"])
def test_append(cuda, dtype, heads_first, tin):
    from warp_b200 import ops
    dt = getattr(torch, dtype)
    ti = dt if tin == "same" else torch.float32
    g = gen(3)
    T, Hq, Hk, D, page, n = 21, 6, 3, 128, 16, 5
    shape = (n, Hk, page, D) if heads_first else (n, page, Hk, D)
    kp = torch.randn(shape, generator=g).to(dt).cuda()
    vp = torch.randn(shape, generator=g).to(dt).cuda()
    if heads_first:
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    x = torch.randn(T, Hq + 2 * Hk, D, generator=g).to(ti).cuda()
    q, k, v = x[:, :Hq], x[:, Hq:Hq + Hk], x[:, Hq + Hk:]
    slots = torch.randperm(n * page, generator=g)[:T].clone()
    slots[4] = slots[9] = -1
    pos = torch.randint(0, 9000, (T,), generator=g, dtype=torch.int32)
    f, _ = ops.rope_inv_freq(64)
    kn = 1 + 0.2 * torch.randn(D, generator=g)
    wk, wv = kp.double().cpu(), vp.double().cpu()
    keep = torch.tensor([t for t in range(T) if slots[t] >= 0])
    wk[slots[keep] // page, slots[keep] % page] = rope64(k.cpu(), pos, f, kn, 1e-6, False,
                                                         1.0)[keep]
    wv[slots[keep] // page, slots[keep] % page] = v.double().cpu()[keep]
    touched = torch.zeros(n, page, dtype=torch.bool)
    touched[slots[keep] // page, slots[keep] % page] = True
    before = kp.clone(), vp.clone()
    qo = ops.kv_append(q, k, v, kp, vp, slots.cuda(), pos.cuda(), f.cuda(), k_norm=kn.cuda())
    assert qo.dtype == dt
    rope_close(qo, rope64(q.cpu(), pos, f, None, 0, False, 1.0))
    rope_close(kp, wk)
    assert torch.equal(vp.cpu(), wv.to(dt))
    for now, was in zip((kp, vp), before):
        assert torch.equal(now[~touched.cuda()], was[~touched.cuda()])
    # keys and values alone leave the same
    kp2, vp2 = (b.clone() for b in before)
    assert ops.kv_append(None, k, v, kp2, vp2, slots.cuda(), pos.cuda(), f.cuda(),
                         k_norm=kn.cuda()) is None
    assert torch.equal(kp2, kp) and torch.equal(vp2, vp)
    ops.attn_status()


def test_append_slot_past_the_pages(cuda):
    from warp_b200 import ffi, ops
    kp = torch.zeros(2, 16, 1, 64, dtype=torch.float16, device="cuda")
    vp = torch.zeros_like(kp)
    k = torch.ones(3, 1, 64, dtype=torch.float16, device="cuda")
    slots = torch.tensor([31, 32, 1 << 40], dtype=torch.int64, device="cuda")
    ops.attn_status()
    ops.kv_append(None, k, k, kp, vp, slots, None, None)
    with pytest.raises(ffi.WarpError, match="slot outside"):
        ops.attn_status()
    ops.attn_status()                       # cleared
    assert vp.sum().item() == 64 and vp[1, 15].sum().item() == 64


def test_slots_plan(cuda):
    from warp_b200 import ops
    q_start = torch.tensor([0, 3, 3, 4, 9], dtype=torch.int32)
    kv_len = torch.tensor([3, 50, 17, 2], dtype=torch.int32)
    pages = torch.tensor([[7, 2, -1], [1, 3, 4], [9, 8, -1], [5, -1, -1]], dtype=torch.int32)
    pos, slots = ops.kv_slots(q_start.cuda(), kv_len.cuda(), pages.cuda(), 16, 11, base=100)
    # request 3 has five queries and two keys: its first three have none
    assert pos.tolist()[:4] == [100, 101, 102, 116]
    assert slots.tolist() == [112, 113, 114, 128, -1, -1, -1, 80, 81, -1, -1]


# ---- attention -----------------------------------------------------------------------


class Case:
    """Ragged requests over shuffled pages; what no request owns is NaN."""

    def __init__(self, q_lens, kv_lens, Hq, Hk, D, page, dtype, heads_first=False, prefix=0,
                 seed=0, sharp=1.0):
        g = gen(seed)
        self.q_lens, self.kv_lens, self.prefix = q_lens, kv_lens, prefix
        B = len(q_lens)
        wide = max(1, max(-(-n // page) for n in kv_lens))
        front = -(-prefix // page)
        total = B * wide + front + 2
        order = torch.randperm(total, generator=g).int()
        self.pages = order[:B * wide].view(B, wide).clone()
        self.pp = order[B * wide:B * wide + front].clone()
        shape = (total, page, Hk, D)
        k, v = (torch.full(shape, math.nan, dtype=torch.float32) for _ in range(2))

        def fill(table, n):
            j = torch.arange(n)
            for x in (k, v):
                x[table[j // page].long(), j % page] = torch.randn(n, Hk, D, generator=g)
        for b, n in enumerate(kv_lens):
            fill(self.pages[b], n)
            self.pages[b, -(-n // page):] = -7          # never looked at
        fill(self.pp, prefix)
        self.k, self.v = k.to(dtype), v.to(dtype)
        self.q = (sharp * torch.randn(sum(q_lens), Hq, D, generator=g)).to(dtype)
        self.page, self.heads_first = page, heads_first
        self.q_start = torch.tensor([0] + q_lens).cumsum(0).int()
        self.kv_len = torch.tensor(kv_lens, dtype=torch.int32)

    def run(self, causal=True, scale=None, q=None, max_q=None, max_kv=None, **kw):
        from warp_b200 import ops

        def place(x):
            if self.heads_first:
                return x.transpose(1, 2).contiguous().cuda().transpose(1, 2)
            return x.cuda()
        out = ops.paged_attention(
            (self.q if q is None else q).cuda(), place(self.k), place(self.v), self.pages.cuda(),
            self.kv_len.cuda(), self.q_start.cuda(),
            max_q=max(self.q_lens) if max_q is None else max_q,
            max_kv=max(self.kv_lens) if max_kv is None else max_kv, scale=scale, causal=causal,
            prefix_pages=self.pp.cuda() if self.prefix else None, prefix_len=self.prefix, **kw)
        ops.attn_status()
        return out.cpu()

    def want(self, causal=True, scale=None):
        """(o, sum p|v| / l) in 64 bits."""
        q, D = self.q.double(), self.q.shape[2]
        scale = 1 / math.sqrt(D) if scale is None else scale
        G = q.shape[1] // self.k.shape[2]
        o, mag = torch.zeros_like(q), torch.zeros_like(q)

        def rows(x, table, n):
            j = torch.arange(n)
            return x[table[j // self.page].long(), j % self.page].double()
        for b, (n, L) in enumerate(zip(self.q_lens, self.kv_lens)):
            t0 = int(self.q_start[b])
            k = torch.cat((rows(self.k, self.pp, self.prefix), rows(self.k, self.pages[b], L)))
            v = torch.cat((rows(self.v, self.pp, self.prefix), rows(self.v, self.pages[b], L)))
            for i in range(n):
                seen = self.prefix + (max(0, min(L, L - n + i + 1)) if causal else L)
                if not seen:
                    continue
                kk, vv = (x[:seen].repeat_interleave(G, 1) for x in (k, v))
                p = (torch.einsum("hd,jhd->hj", q[t0 + i], kk) * scale).softmax(-1)
                o[t0 + i] = torch.einsum("hj,jhd->hd", p, vv)
                mag[t0 + i] = torch.einsum("hj,jhd->hd", p, vv.abs())
        return o, mag

    def check(self, **kw):
        got = self.run(**kw)
        o, mag = self.want(**{k: v for k, v in kw.items() if k in ("causal", "scale")})
        u = ROUND[got.dtype]
        tol = 2 * (u * o.abs() + (u + 2.0 ** -14) * mag)
        bad = ~((got.double() - o).abs() <= tol)
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3],
                               (got.double() - o).abs().max().item())
        return got


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq, Hk", [(1, 1), (4, 4), (18, 2), (56, 8), (16, 1), (40, 1), (12, 4)])
def test_decode(cuda, dtype, D, Hq, Hk):
    """One token a request: no key, one, around a tile and a page, many."""
    kv = [1, 0, 15, 16, 17, 31, 33, 300, 1025]
    Case([1] * len(kv), kv, Hq, Hk, D, 16, dtype, seed=Hq).check()


@pytest.mark.parametrize("page, heads_first", [(16, True), (32, False), (64, True), (128, False),
                                               (1024, False), (4096, True)])
def test_decode_pages(cuda, page, heads_first):
    Case([1] * 4, [5, 130, 1000, 4097 if page < 4096 else 129], 8, 2, 128, page, torch.bfloat16,
         heads_first, seed=page).check()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("L", [4095, 20001])
def test_decode_long(cuda, D, L):
    """Few requests over long ranges: parts of the range, joined."""
    Case([1, 1], [L, 3], 14, 2, D, 64, torch.bfloat16, seed=5, sharp=2.0).check()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q, kv", [([2], [2]), ([3, 1, 5], [3, 9, 40]), ([17], [17]),
                                   ([33, 1, 64], [33, 200, 64]), ([130], [130]),
                                   ([129, 2, 70], [400, 2, 71]), ([1, 257], [1500, 900])])
def test_chunks(cuda, dtype, D, q, kv):
    Case(q, kv, 6, 2, D, 16, dtype, seed=sum(q)).check()


@pytest.mark.parametrize("Hq, Hk", [(1, 1), (7, 1), (9, 3), (32, 1), (130, 1)])
def test_chunk_heads(cuda, Hq, Hk):
    Case([40, 7], [90, 7], Hq, Hk, 128, 32, torch.bfloat16, seed=Hq).check()


@pytest.mark.parametrize("q, kv", [([1, 1], [0, 77]), ([5, 2], [3, 300]), ([150], [61]),
                                   ([4, 90, 3], [0, 0, 1])])
def test_not_causal(cuda, q, kv):
    """Every query sees every key, as in cross attention; no key gives zeros."""
    c = Case(q, kv, 8, 4, 64, 16, torch.float16, seed=9)
    got = c.check(causal=False)
    for b, L in enumerate(kv):
        if not L:
            assert not got[int(c.q_start[b]):int(c.q_start[b + 1])].any()


@pytest.mark.parametrize("q, kv", [([5], [2]), ([40, 3], [33, 1]), ([200], [100]), ([2, 1], [0, 4])])
def test_more_queries_than_keys(cuda, q, kv):
    """Causal rows before the first key are empty: zeros."""
    c = Case(q, kv, 8, 2, 128, 16, torch.bfloat16, seed=11)
    got = c.check()
    assert not got[:q[0] - kv[0]].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("prefix", [1, 16, 100, 515, 3001])
def test_prefix_decode(cuda, dtype, D, prefix):
    Case([1] * 5, [1, 40, 0, 16, 333], 18, 2, D, 16, dtype, prefix=prefix, seed=prefix).check()


@pytest.mark.parametrize("q, kv, prefix", [
    ([1], [7], 300),                        # one request: nothing to share
    ([3, 2, 5], [3, 2, 9], 70),             # few tokens each
    ([100, 90], [100, 95], 130),            # rows enough of their own
    ([1, 300, 1], [5, 300, 2], 64),         # mixed
    ([1] * 40, [2] * 40, 200)])
@pytest.mark.parametrize("causal", [True, False])
def test_prefix_shapes(cuda, q, kv, prefix, causal):
    Case(q, kv, 8, 2, 128, 32, torch.bfloat16, prefix=prefix, seed=len(q)).check(causal=causal)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B, Hq, Hk", [(2, 4, 4), (3, 10, 2), (16, 2, 2), (17, 2, 2)])
@pytest.mark.parametrize("prefix", [5, 333, 2600])
def test_prefix_few_rows(cuda, dtype, D, B, Hq, Hk, prefix):
    """All the batch's rows of a kv head in one tile of 16, and one more."""
    Case([1] * B, [i * 7 % 40 for i in range(B)], Hq, Hk, D, 16, dtype, prefix=prefix,
         seed=B + prefix).check()


def test_one_page_and_one_head(cuda):
    """Axes of one entry, whose strides mean nothing."""
    for n in (1, 40):
        c = Case([n], [60], 2, 1, 64, 64, torch.float16, seed=28)
        at = c.pages[0, :1].long()
        c.k, c.v, c.pages = c.k[at], c.v[at], torch.zeros(1, 1, dtype=torch.int32)
        c.check()


def test_prefix_is_the_same_as_its_own_copy(cuda):
    """A shared prefix gives what the same keys at the head of each request's own pages give."""
    P, own = 96, [5, 33]
    c = Case([1, 1], own, 8, 2, 64, 16, torch.float16, prefix=P, seed=21)
    d = Case([1, 1], [P + n for n in own], 8, 2, 64, 16, torch.float16, seed=22)
    d.q = c.q
    for b, n in enumerate(own):
        for x, y in ((c.k, d.k), (c.v, d.v)):
            j = torch.arange(P + n)
            at = d.pages[b][j // 16].long(), j % 16
            y[at] = torch.cat((x[c.pp[j[:P] // 16].long(), j[:P] % 16],
                               x[c.pages[b][j[:n] // 16].long(), j[:n] % 16]))
    want, mag = c.want()
    assert torch.equal(want, d.want()[0])
    for x in (c.run(), d.run()):
        assert ((x.double() - want).abs() <= 4 * (2.0 ** -11 + 2.0 ** -14) * mag).all()


@pytest.mark.parametrize("sharp, scale", [(0.0, None), (30.0, None), (1.0, 1e-4), (1.0, 2.0)])
def test_flat_and_sharp_rows(cuda, sharp, scale):
    for q, kv in (([1, 1], [700, 90]), ([150], [400])):
        Case(q, kv, 8, 2, 128, 64, torch.bfloat16, seed=13, sharp=sharp).check(scale=scale)


def test_rising_scores(cuda):
    """Each key outdoes those before it, so that the running maximum always moves."""
    for q, kv in (([1], [900]), ([140], [700])):
        c = Case(q, kv, 4, 1, 128, 64, torch.bfloat16, seed=14)
        j = torch.arange(kv[0])
        c.q[:] = 1.0
        c.k[c.pages[0][j // 64].long(), j % 64] = (j * 0.02)[:, None, None].to(torch.bfloat16)
        c.check()


@pytest.mark.parametrize("n", [6, 20, 150])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_later_values_that_are_not_finite(cuda, n, value):
    """A value behind a row's last key does not reach it, whatever it is; a
    value in sight does."""
    L, at = n + 9, n + 9 - n // 2
    c = Case([n], [L], 6, 2, 128, 16, torch.bfloat16, seed=15)
    want, mag = c.want()
    c.v[c.pages[0][at // 16].long(), at % 16, 1, 70] = value
    got = c.run()
    first = at - (L - n)                    # the first query that sees key `at`
    sees = torch.zeros(n, 6, 128, dtype=torch.bool)
    sees[first:, 3:, 70] = True
    tol = 2 * (2.0 ** -9 * want.abs() + (2.0 ** -9 + 2.0 ** -14) * mag)
    assert ((got.double() - want).abs() <= tol)[~sees].all()
    hit = got[sees]
    assert hit.isnan().all() if math.isnan(value) else (hit == value).all()


def test_masked_keys_that_are_not_finite(cuda):
    """A later key's NaN has no effect on a row that does not see it."""
    for n in (6, 150):
        c = Case([n], [n], 4, 2, 64, 16, torch.float16, seed=16)
        want = c.run()
        c.k[c.pages[0][(n - 1) // 16].long(), (n - 1) % 16] = math.nan
        got = c.run()
        assert torch.equal(got[:-1], want[:-1]) and got[-1].isnan().all()


def test_strided_queries_and_given_out(cuda):
    from warp_b200 import ops
    c = Case([1, 3], [50, 20], 8, 2, 64, 16, torch.float16, seed=17)
    wide = torch.full((4, 3, 8, 80), math.nan, dtype=torch.float16)
    wide[:, 1, :, 8:72] = c.q
    q = wide.cuda()[:, 1, :, 8:72]
    out = torch.empty(4, 8, 64, dtype=torch.float16, device="cuda")
    want = c.run()
    got = ops.paged_attention(q, c.k.cuda(), c.v.cuda(), c.pages.cuda(), c.kv_len.cuda(),
                              c.q_start.cuda(), 3, 50, out=out)
    assert got is out and torch.equal(got.cpu(), want)


def test_loose_bounds_give_the_same_within_tolerance(cuda):
    """Larger host bounds only change how the work is cut."""
    c = Case([1, 2, 1], [200, 31, 7], 8, 2, 64, 16, torch.bfloat16, seed=18)
    c.pages = torch.cat((c.pages, torch.full((3, 40), -7, dtype=torch.int32)), 1)
    c.check()
    c.check(max_q=64, max_kv=13 * 16 + 500)


def test_bounds_are_reported(cuda):
    from warp_b200 import ffi, ops
    c = Case([1, 2], [200, 31], 8, 2, 64, 16, torch.bfloat16, seed=19)
    ops.attn_status()
    with pytest.raises(ffi.WarpError, match="length"):
        c.run(max_kv=100)
    with pytest.raises(ffi.WarpError, match="length"):
        c.run(max_q=1)
    c.pages[0, 3] = 10 ** 6
    with pytest.raises(ffi.WarpError, match="page number"):
        c.run()
    c.pages[0, 3] = -1
    with pytest.raises(ffi.WarpError, match="page number"):
        c.run()
    ops.attn_status()


def test_same_bits_every_time_and_on_another_stream(cuda):
    c = Case([1, 1, 3], [3000, 50, 700], 14, 2, 128, 64, torch.bfloat16, prefix=333, seed=20)
    want = c.run()
    for _ in range(3):
        assert torch.equal(c.run(), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = c.run()
    assert torch.equal(got, want)


def test_captured_step(cuda):
    """slots, append and attention in one graph; lengths move between replays."""
    from warp_b200 import ops
    g = gen(23)
    B, Hq, Hk, D, page = 3, 8, 2, 64, 16
    kp = torch.zeros(20, page, Hk, D, dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros_like(kp)
    pages = torch.randperm(20, generator=g)[:12].view(B, 4).int().cuda()
    q_start = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    kv_len = torch.tensor([0, 5, 30], dtype=torch.int32, device="cuda")
    x = torch.zeros(B, Hq + 2 * Hk, D, device="cuda")
    f, _ = ops.rope_inv_freq(D, device="cuda")

    def step():
        pos, slots = ops.kv_slots(q_start, kv_len, pages, page, B)
        q = ops.kv_append(x[:, :Hq], x[:, Hq:Hq + Hk], x[:, Hq + Hk:], kp, vp, slots, pos, f)
        return ops.paged_attention(q, kp, vp, pages, kv_len, q_start, 1, 64)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    kp.zero_(), vp.zero_()
    kk, vv = [[] for _ in range(B)], [[] for _ in range(B)]
    for b, n in enumerate((0, 5, 30)):      # what was there before: zeros
        kk[b] += [torch.zeros(Hk, D, dtype=torch.float64)] * n
        vv[b] += [torch.zeros(Hk, D, dtype=torch.float64)] * n
    for n in range(20):
        xs = torch.randn(B, Hq + 2 * Hk, D, generator=g)
        x.copy_(xs)
        kv_len += 1
        graph.replay()
        torch.cuda.synchronize()
        for b in range(B):
            pos = torch.tensor([len(kk[b])])
            r = rope64(xs[b:b + 1, :Hq + Hk], pos, f.cpu(), None, 0, False, 1.0)[0]
            kk[b].append(r[Hq:].to(torch.bfloat16).double())
            vv[b].append(xs[b, Hq + Hk:].to(torch.bfloat16).double())
            k, v = (torch.stack(z).repeat_interleave(Hq // Hk, 1) for z in (kk[b], vv[b]))
            q = r[:Hq].to(torch.bfloat16).double()
            p = (torch.einsum("hd,jhd->hj", q, k) / 8).softmax(-1)
            o, mag = torch.einsum("hj,jhd->hd", p, v), torch.einsum("hj,jhd->hd", p, v.abs())
            # a rotated value whose rounding falls the other way moves scores
            # by up to u |q||k| / 8, so weights by a few u
            err = (out[b].double().cpu() - o).abs()
            assert (err <= 2.0 ** -8 * o.abs() + 2.0 ** -6 * mag).all(), (n, b)
    ops.attn_status()
    del graph


def test_long_cache_offsets(cuda):
    """Pages whose offsets pass 2^31 elements."""
    from warp_b200 import ops
    page, Hk, D = 4096, 8, 128
    n = 2 ** 31 // (page * Hk * D) + 8      # 520 pages, 4.4 GB each of K and V
    kp = torch.zeros(n, page, Hk, D, dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros_like(kp)
    pages = torch.tensor([[n - 1, 0, n - 2]], dtype=torch.int32, device="cuda")
    L = 2 * page + 100
    k = torch.randn(L, Hk, D, generator=gen(24)).bfloat16().cuda()
    v = torch.randn(L, Hk, D, generator=gen(25)).bfloat16().cuda()
    q_start = torch.tensor([0, L], dtype=torch.int32, device="cuda")
    kv_len = torch.tensor([L], dtype=torch.int32, device="cuda")
    pos, slots = ops.kv_slots(q_start, kv_len, pages, page, L)
    ops.kv_append(None, k, v, kp, vp, slots, None, None)
    assert torch.equal(kp[n - 2, :100], k[2 * page:]) and torch.equal(vp[n - 1], v[:page])
    q = torch.randn(1, Hk, D, generator=gen(26)).bfloat16().cuda()
    one = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    got = ops.paged_attention(q, kp, vp, pages, kv_len, one, 1, L)
    p = (torch.einsum("hd,jhd->hj", q[0].double(), k.double()) / math.sqrt(D)).softmax(-1)
    o = torch.einsum("hj,jhd->hd", p, v.double())
    mag = torch.einsum("hj,jhd->hd", p, v.double().abs())
    assert ((got[0].double() - o).abs() <= 2 * (2.0 ** -9 * o.abs() + 2.0 ** -8 * mag)).all()
    ops.attn_status()


def test_wrapper_refusals(cuda):
    from warp_b200 import ffi, ops
    c = Case([1], [20], 4, 2, 64, 16, torch.float16)
    k, v = c.k.cuda(), c.v.cuda()
    args = (c.pages.cuda(), c.kv_len.cuda(), c.q_start.cuda(), 1, 20)
    q = c.q.cuda()
    with pytest.raises(ffi.WarpError, match="type"):
        ops.paged_attention(q.bfloat16(), k, v, *args)
    with pytest.raises(ffi.WarpError, match="over"):
        ops.paged_attention(q[:, :3], k, v, *args)
    with pytest.raises(ValueError, match="out must"):
        ops.paged_attention(q, k, v, *args, out=q.float())
    with pytest.raises(ValueError, match="prefix_pages"):
        ops.paged_attention(q, k, v, *args, prefix_pages=c.pages.cuda()[0], prefix_len=33)
    with pytest.raises(ValueError, match="contiguous"):
        ops.paged_attention(q.transpose(1, 2).contiguous().transpose(1, 2), k, v, *args)
    with pytest.raises(ValueError, match="pages must"):
        ops.paged_attention(q, k, v, c.pages.cuda().long(), *args[1:])
    with pytest.raises(ValueError, match="kv_len"):
        ops.paged_attention(q, k, v, args[0], args[1].long(), *args[2:])
    with pytest.raises(ffi.WarpError, match="page_size"):
        ops.paged_attention(q, k[:, :8], v[:, :8], *args)
    f, _ = ops.rope_inv_freq(64, device="cuda")
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(ffi.WarpError, match="type"):
        ops.qk_norm_rope(q, None, pos, f, out_dtype=torch.float32)
    with pytest.raises(ValueError, match="positions"):
        ops.qk_norm_rope(q, None, pos.long(), f)
    with pytest.raises(ValueError, match="inv_freq"):
        ops.qk_norm_rope(q, None, pos, f.float())
    with pytest.raises(ValueError, match="q_norm"):
        ops.qk_norm_rope(q, None, pos, f, q_norm=torch.ones(32, device="cuda"))
    with pytest.raises(ValueError, match="slots"):
        ops.kv_append(None, q[:, :2], q[:, :2], k, v, pos, pos, f)
    with pytest.raises(ffi.WarpError, match="heads"):
        ops.kv_append(None, q, q, k, v, pos.long(), pos, f)


def test_scores_of_minus_infinity(cuda):
    """Keys that score -inf weigh nothing, and a row with no other score gives zeros."""
    for n, L in ((1, 300), (150, 300)):
        c = Case([n], [L], 4, 2, 64, 16, torch.float16, seed=27)
        c.q[..., 0] = 1.0
        want_all = c.k.clone()
        j = torch.arange(L)
        at = c.pages[0][j // 16].long(), j % 16
        c.k[at[0], at[1], 0, 0] = -math.inf         # kv head 0: every key
        c.k[at[0][1::2], at[1][1::2], 1, 0] = -math.inf     # kv head 1: every other
        got = c.run(causal=False)
        assert not got[:, :2].any()
        c.k = want_all
        keep = c.k[at][0::2], c.v[at][0::2]
        for h in (2, 3):
            p = (c.q[:, h].double() @ keep[0][:, 1].double().T / 8).softmax(-1)
            o, mag = p @ keep[1][:, 1].double(), p @ keep[1][:, 1].double().abs()
            tol = 2 * (2.0 ** -11 * o.abs() + (2.0 ** -11 + 2.0 ** -14) * mag)
            assert ((got[:, h].double() - o).abs() <= tol).all()
