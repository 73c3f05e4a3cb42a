"""The decoder block: attention over a paged cache and the MoE layer in one
path, prompts and single tokens, with and without a shared prefix.

The attention half is checked against 64-bit arithmetic on the dequantised
weights.  What it rounds: k, v and q to the pages' type, the softmax's weights,
the result (each u = 2^-9 of bf16), and the trunk's fp32 products.  Scores move
by a few u * |q||k| / sqrt(D), of order u for normed heads, so the half as a
whole is within some 8 u of its norm."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HIDDEN, HQ, HK, D, PAGE = 512, 6, 2, 64, 16
TOL = 8 * 2.0 ** -9


def trunk(rows, cols, seed, bits=4):
    """(device matrix, the same in 64 bits)."""
    from warp_b200 import synth
    from warp_b200.block import Trunk
    W = torch.randn(rows, cols, generator=torch.Generator().manual_seed(seed)) * 0.05
    w, s = synth.quantize_q(W, 32, bits)
    if bits == 4:
        q = torch.stack((w & 15, w >> 4), -1).view(rows, cols).double() - 8
    else:
        q = w.view(torch.int8).double()
    exact = (q.view(rows, -1, 32) * s.view(torch.float16).double()[..., None]).view(rows, cols)
    return Trunk(w.cuda(), s.cuda(), rows, cols, 32, bits), exact


@pytest.fixture(scope="module")
def made(cuda):
    from warp_b200 import ops, synth
    from warp_b200.block import DecoderBlock
    bank = synth.random_bank(16, HIDDEN, 256, seed=1, device=cuda)
    layer = synth.SyntheticLayer(bank, synth.router_matrix(16, HIDDEN, 2, device=cuda),
                                 synth.shared_expert(HIDDEN, 256, 3, device=cuda))
    moe = layer.moe(4, max_tokens=8, prefill_tokens=256)
    g = torch.Generator().manual_seed(4)
    qkv, qkv64 = trunk((HQ + 2 * HK) * D, HIDDEN, 5)
    proj, proj64 = trunk(HIDDEN, HQ * D, 6, bits=8)
    n1, n2 = (1 + 0.1 * torch.randn(HIDDEN, generator=g) for _ in range(2))
    qn, kn = (1 + 0.1 * torch.randn(D, generator=g) for _ in range(2))
    f, s = ops.rope_inv_freq(D, scaling="yarn", factor=4.0, trained=64)
    block = DecoderBlock(moe, qkv, proj, HQ, HK, D, n1.cuda(), n2.cuda(), f.cuda(), s, qn.cuda(),
                         kn.cuda())
    return block, dict(qkv=qkv64, proj=proj64, n1=n1, qn=qn, kn=kn, f=f, s=s)


def cache(pages, dtype):
    nan = float("nan")
    return tuple(torch.full((pages, PAGE, HK, D), nan, dtype=dtype, device="cuda")
                 for _ in range(2))


def attend64(m, seqs):
    """The attention half over whole sequences, [n][hidden] each, in 64 bits."""
    def norm(x, w):
        return x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.double()

    def turn(x):
        a = torch.arange(x.shape[0]).double()[:, None] * m["f"]
        c, s = torch.cos(a)[:, None] * m["s"], torch.sin(a)[:, None] * m["s"]
        lo, hi = x[..., :D // 2], x[..., D // 2:]
        return torch.cat((lo * c - hi * s, lo * s + hi * c), -1)
    out = []
    for h in seqs:
        h = h.double()
        x = (norm(h, m["n1"]) @ m["qkv"].T).view(-1, HQ + 2 * HK, D)
        q, k = turn(norm(x[:, :HQ], m["qn"])), turn(norm(x[:, HQ:HQ + HK], m["kn"]))
        k, v = (z.repeat_interleave(HQ // HK, 1) for z in (k, x[:, HQ + HK:]))
        p = torch.einsum("thd,jhd->htj", q, k) / 8
        p = p.masked_fill(torch.ones(p.shape[1:]).triu(1).bool(), -torch.inf).softmax(-1)
        out.append(h + torch.einsum("htj,jhd->thd", p, v).reshape(len(h), -1) @ m["proj"].T)
    return out


def rel(a, b):
    return ((a.double().cpu() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompts_then_tokens(made, dtype):
    """Ragged prompts in one step, then tokens one by one, against whole sequences."""
    from warp_b200 import ops
    from warp_b200.block import Step
    block, m = made
    lens, more = [70, 3, 25], 4
    g = torch.Generator().manual_seed(7)
    seqs = [torch.randn(n + more, HIDDEN, generator=g) for n in lens]
    want = attend64(m, seqs)
    pages = torch.randperm(3 * 5, generator=g).int().view(3, 5).cuda()
    kp, vp = cache(15, dtype)

    def step(new, upto):
        s = Step.plan(new, upto, pages, PAGE)
        h = torch.cat([x[n - k:n] for x, n, k in zip(seqs, upto, new)]).cuda()
        # attend first, then the whole block over the same slots
        got = block.attend(h, kp, vp, s)
        w = torch.cat([x[n - k:n] for x, n, k in zip(want, upto, new)])
        assert rel(got, w) < TOL
        out = block.forward(h, kp, vp, s)
        if sum(new) <= block.moe.max_tokens:
            moe = block.moe.forward_block(got, torch.empty_like(got), block.norm2, block.eps)
        else:
            moe = block.moe.prefill(ops.rmsnorm(got, block.norm2, block.eps), residual=got)
        assert torch.equal(out, moe)
        block.moe.status()
    step(lens, lens)
    for i in range(1, more + 1):
        step([1] * 3, [n + i for n in lens])
    ops.attn_status()


def test_shared_prefix(made):
    """Tokens behind a prefix that one request put into the pages, against whole sequences."""
    from warp_b200 import ops
    from warp_b200.block import Step
    block, m = made
    g = torch.Generator().manual_seed(8)
    P, own = 37, [1, 18, 5]
    head = torch.randn(P, HIDDEN, generator=g)
    tails = [torch.randn(n, HIDDEN, generator=g) for n in own]
    want = attend64(m, [torch.cat((head, t)) for t in tails])
    kp, vp = cache(12, torch.bfloat16)
    front = torch.tensor([[9, 2, 5]], dtype=torch.int32, device="cuda")
    block.attend(head.cuda(), kp, vp, Step.plan([P], [P], front, PAGE))
    pages = torch.tensor([[0, 1], [3, 4], [6, 7]], dtype=torch.int32, device="cuda")
    for new, upto in ((own[:], own),):
        s = Step.plan(new, upto, pages, PAGE, prefix_pages=front[0], prefix_len=P)
        got = block.attend(torch.cat(tails).cuda(), kp, vp, s)
        assert rel(got, torch.cat([w[P:] for w in want])) < TOL
    ops.attn_status()


def test_refuses_what_does_not_fit(made):
    from warp_b200.block import DecoderBlock, Step
    block, _ = made
    with pytest.raises(ValueError, match="projections"):
        DecoderBlock(block.moe, block.qkv, block.proj, HQ, HK + 1, D, block.norm1, block.norm2,
                     block.inv_freq)
    with pytest.raises(ValueError, match="requests"):
        Step.plan([1, 2], [3], torch.zeros(2, 1, dtype=torch.int32, device="cuda"), PAGE)
