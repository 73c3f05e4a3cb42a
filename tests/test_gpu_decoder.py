"""Whole steps of drafted tokens, as they are used: plan, blocks over the paged
caches, head, pick, accept, one after another with requests that grow and end.

Greedy decoding token by token is the measure.  A step of several tokens takes its
trunk products, experts and attention through other kernels than a step of one
(bf16 and fp16 operands, rounded weights), so its logits are off by some hundredths of their
deviation; choices are compared as long as the best token leads by more than that."""
import pytest
import torch

from test_gpu_block import D, HIDDEN, HK, HQ, PAGE, trunk

pytestmark = pytest.mark.gpu

V, LAYERS, WIDE = 1000, 2, 8
LEAD = 0.1                                  # of the logits' deviation


def starts(lengths):
    return torch.tensor([0] + lengths).cumsum(0).int().cuda()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.fixture(scope="module")
def model(cuda):
    from warp_b200 import ops, synth
    from warp_b200.block import DecoderBlock
    g = torch.Generator().manual_seed(21)
    blocks = []
    for i in range(LAYERS):
        bank = synth.random_bank(8, HIDDEN, 256, seed=30 + i, device=cuda)
        layer = synth.SyntheticLayer(bank, synth.router_matrix(8, HIDDEN, 40 + i, device=cuda),
                                     synth.shared_expert(HIDDEN, 256, 50 + i, device=cuda))
        n1, n2 = (1 + 0.1 * torch.randn(HIDDEN, generator=g) for _ in range(2))
        f, s = ops.rope_inv_freq(D)
        blocks.append(DecoderBlock(layer.moe(2, max_tokens=8, prefill_tokens=256),
                                   trunk((HQ + 2 * HK) * D, HIDDEN, 60 + i)[0],
                                   trunk(HIDDEN, HQ * D, 70 + i)[0], HQ, HK, D, n1.cuda(),
                                   n2.cuda(), f.cuda(), s))
    embed = torch.randn(V, HIDDEN, generator=g).cuda()
    return blocks, embed, torch.ones(HIDDEN, device="cuda"), trunk(V, HIDDEN, 80, bits=8)[0]


def decoder(model, requests, pages, dtype=torch.bfloat16):
    from warp_b200.block import Decoder
    shape = (LAYERS, pages, PAGE, HK, D)
    k, v = (torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    return Decoder(*model, k, v, requests, WIDE)


def greedy(model, prompt, n):
    """n tokens one by one, and by how much of the logits' deviation each led."""
    from warp_b200 import ops
    d = decoder(model, 1, WIDE)
    heard, inner = [], d._logits

    def logits(h):
        heard.append(inner(h))
        return heard[-1]
    d._logits = logits
    tokens = [int(d.extend(i32(prompt), starts([len(prompt)]), len(prompt)))]
    while len(tokens) < n:
        tokens.append(int(d.extend(i32(tokens[-1:]), starts([1]), 1)))
    ops.attn_status()
    lead = []
    for x in heard:
        top = x[-1].topk(2).values
        lead.append(float((top[0] - top[1]) / x[-1].std()))
    return tokens, lead


def test_extend_is_the_plain_step(model):
    """A prompt through the decoder against the blocks driven by a step from the host."""
    from warp_b200 import ops
    from warp_b200.block import Step
    g = torch.Generator().manual_seed(1)
    lens = [20, 1, 33]
    tokens = torch.randint(0, V, (sum(lens),), generator=g, dtype=torch.int32).cuda()
    d = decoder(model, 3, 3 * WIDE)
    got = d.extend(tokens, starts(lens), max(lens))
    pages = torch.arange(3 * WIDE, dtype=torch.int32, device="cuda").view(3, WIDE)
    k, v = torch.zeros_like(d.k_pages), torch.zeros_like(d.v_pages)
    step, h = Step.plan(lens, lens, pages, PAGE), d.embed[tokens]
    for block, kl, vl in zip(d.blocks, k, v):
        h = block.forward(h, kl, vl, step)
    want = ops.pick_tokens(d._logits(h[starts(lens)[1:].long() - 1]))
    ops.attn_status()
    assert torch.equal(got, want)
    assert d.kv_len.tolist() == lens and d.held.tolist() == [-(-n // PAGE) for n in lens]


@pytest.mark.parametrize("right", ["all", "some", "none"])
def test_drafted_steps_are_greedy_decoding(model, right):
    """Requests of unequal length decode with trees of which one branch is right for a
    while; what they choose is what they would have chosen one by one."""
    from warp_b200 import ops
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, V, (n,), generator=g).tolist() for n in (37, 5, 16)]
    n = 14
    true = [greedy(model, p, n) for p in prompts]
    d = decoder(model, 3, 3 * WIDE - 4)
    lens = [len(p) for p in prompts]
    first = d.extend(i32(sum(prompts, [])), starts(lens), max(lens)).tolist()
    done = [[t] for t in first]
    steps = 0
    while min(map(len, done)) < n - 4:
        drafted, parents, sizes = [], [], []
        for b in range(3):
            at = len(done[b])
            after = (true[b][0] + [1] * 8)[at:at + 3]
            if right == "none" or (right == "some" and steps % 2 == b % 2):
                after = [(t + 1) % V for t in after]
            # node 0, a wrong branch, the right one behind it, and wrong leaves
            tree = [done[b][-1], (after[0] + 7) % V, after[0], (after[1] + 5) % V, after[1],
                    after[2], 3]
            up = [-1, 0, 0, 1, 2, 4, 4]
            if b == 1:
                tree, up = tree[:5], up[:5]
            drafted, parents, sizes = drafted + tree, parents + up, sizes + [len(tree)]
        count, chosen = d.verify(i32(drafted), i32(parents), starts(sizes), max(sizes))
        for b, c in enumerate(count.tolist()):
            assert 1 <= c <= 4
            done[b] += chosen[b, :c].tolist()
        steps += 1
    ops.attn_status()
    for (want, lead), got in zip(true, done):
        sure = next((i for i, x in enumerate(lead) if x < LEAD), n)
        m = min(sure, len(got), n)
        assert got[:m] == want[:m]
    # keys: the prompt and all certain tokens but the last; pages to hold them and the trees
    assert d.kv_len.tolist() == [a + len(t) - 1 for a, t in zip(lens, done)]
    if right == "all":
        assert steps < n - 5


def test_pages_of_requests_that_end(model):
    """A pool that holds two requests serves one after another."""
    from warp_b200 import ops
    d = decoder(model, 3, 2 * WIDE)
    prompt = i32(list(range(100)))
    for turn in range(4):
        lens = [100 if b == turn % 3 else 0 for b in range(3)]
        d.extend(prompt, starts(lens), 100)
        ops.attn_status()
        assert d.held[turn % 3] == -(-100 // PAGE)
        d.kv_len[turn % 3] = 0
    d.extend(prompt[:3], starts([1, 1, 1]), 1)
    ops.attn_status()
    assert d.held.tolist() == [1, 1, 1] and d.pool[0] == 2 * WIDE - 3


def test_a_captured_step_replays(model):
    """Trees of a fixed shape as one graph: padding nodes are never accepted, lengths and
    pages move on from replay to replay as without a graph."""
    from warp_b200 import ops
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, V, (n,), generator=g).tolist() for n in (9, 30)]
    parents, q_start = i32([-1, 0, 0, 2, -1, 0, 0, 2]), starts([4, 4])

    def start():
        d = decoder(model, 2, 2 * WIDE)
        lens = [len(p) for p in prompts]
        return d, d.extend(i32(sum(prompts, [])), starts(lens), max(lens))

    def step(d):
        count, chosen = d.verify(drafted, parents, q_start, 4)
        drafted[0::4] = chosen.gather(1, (count - 1)[:, None].long())[:, 0]
        return count, chosen
    # the trunk's matmul wants a call on the stream before it is captured
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        d, first = start()
        drafted = torch.full((8,), -1, dtype=torch.int32, device="cuda")
        drafted[0::4] = first
        plain = []
        for _ in range(5):
            count, chosen = step(d)
            plain.append((count.tolist(), chosen.tolist()))
        end = d.kv_len.tolist()
        d, again = start()
        assert torch.equal(first, again)
        drafted[0::4] = first
        kept = [x.clone() for x in (d.kv_len, d.held, d.pages, d.pool, drafted)]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            count, chosen = step(d)
        for x, y in zip((d.kv_len, d.held, d.pages, d.pool, drafted), kept):
            assert torch.equal(x, y)        # capturing runs nothing
        for want in plain:
            graph.replay()
            assert (count.tolist(), chosen.tolist()) == want
        assert d.kv_len.tolist() == end
    ops.attn_status()


def test_choices_are_weighed(model):
    """Masks and biases reach every node of a step."""
    d = decoder(model, 1, WIDE)
    first = d.extend(i32([1, 2, 3]), starts([3]), 3)
    only = torch.zeros((V + 31) // 32, dtype=torch.int32)
    only[7] = 1 << 5                        # token 229 alone
    count, chosen = d.verify(torch.cat((first, i32([229, 229, 5]))), i32([-1, 0, 1, 1]),
                             starts([4]), 4, allowed=only.cuda())
    assert count.tolist() == [3] and chosen.tolist() == [[229, 229, 229, -1]]
    bias = torch.zeros(V, device="cuda")
    bias[11] = 1e4
    count, chosen = d.verify(i32([229, 11]), i32([-1, 0]), starts([2]), 2, bias=bias)
    assert count.tolist() == [2] and chosen.tolist() == [[11, 11]]


def test_numbers_outside_the_vocabulary(model):
    """They are no fault: a drafted one is never accepted, a start out of place is said."""
    from warp_b200 import ops
    d = decoder(model, 1, WIDE)
    first = d.extend(i32([V + 5, -1, 1 << 30]), starts([3]), 3)
    again = decoder(model, 1, WIDE).extend(i32([V - 1, 0, V - 1]), starts([3]), 3)
    assert torch.equal(first, again)
    count, chosen = d.verify(torch.cat((first, i32([V, 1 << 30, -1]))), i32([-1, 0, 1, 0]),
                             starts([4]), 4)
    ops.attn_status()
    assert count.tolist() == [1] and 0 <= chosen[0, 0] < V and d.kv_len.tolist() == [4]


def test_steps_that_are_refused(model):
    """Before anything is done, or with the requests as they were."""
    d = decoder(model, 2, WIDE)
    for call in (lambda: d.extend(i32([]), i32([0, 0, 0]), 1),
                 lambda: d.verify(i32([]), i32([]), i32([0, 0, 0]), 1),
                 lambda: d.extend(i32([1, 2]), i32([0, 2]), 2),
                 lambda: d.verify(i32([1, 2]), i32([-1]), i32([0, 1, 2]), 1),
                 lambda: d.extend(i32([1, 2]), i32([0, 1, 2]), 1, bias=torch.zeros(V - 1).cuda())):
        with pytest.raises(ValueError):
            call()
        assert d.kv_len.tolist() == [0, 0]
