"""Steps of a decoder whose pool runs empty: a request without pages for all its keys stays as
it was, the others go on, and it goes on itself when there are pages again."""
import pytest
import torch

from test_gpu_block import PAGE
from test_gpu_decoder import V, WIDE, decoder, i32, model, starts  # noqa: F401

pytestmark = pytest.mark.gpu


def tokens(seed, n):
    return torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(seed),
                         dtype=torch.int32).cuda()


def starved():
    from warp_b200 import ffi, ops
    with pytest.raises(ffi.WarpError, match="no page left"):
        ops.attn_status()


def tree_of(first, other):
    """Two nodes behind node 0, and one behind the second."""
    return torch.cat((first.view(1), i32(other)))


UP = [-1, 0, 0, 2]


def test_a_prompt_without_pages_waits(model):  # noqa: F811
    """Of two prompts the second gets too few pages; when the first request ends, the same
    prompt again gives what it gives alone."""
    from warp_b200 import ops
    ops.attn_status()
    a, b = tokens(1, 5 * PAGE - 3), tokens(2, 4 * PAGE - 7)
    lens = [len(a), len(b)]
    whole, d = decoder(model, 2, 2 * WIDE), decoder(model, 2, 7)
    want = whole.extend(torch.cat((a, b)), starts(lens), max(lens))
    ops.attn_status()
    got = d.extend(torch.cat((a, b)), starts(lens), max(lens))
    starved()
    assert got.tolist() == [want[0].item(), -1]
    assert d.kv_len.tolist() == [len(a), 0] and d.held.tolist() == [5, 2]
    # the first goes on while the second has too few still
    step = (i32([got[0].item()]), starts([1, 0]), 1)
    assert d.extend(*step)[0] == whole.extend(*step)[0]
    ops.attn_status()
    assert d.kv_len.tolist() == [len(a) + 1, 0] and d.held.tolist() == [5, 0]
    # it ends, and its pages are what the second needs
    d.kv_len[0] = 0
    alone = decoder(model, 2, 2 * WIDE)
    step = (b, starts([0, len(b)]), len(b))
    assert d.extend(*step)[1] == alone.extend(*step)[1]
    ops.attn_status()
    assert d.kv_len.tolist() == [0, len(b)] and d.held.tolist() == [0, 4]


def test_a_tree_without_pages_waits(model):  # noqa: F811
    """A step of drafted tokens that needs a page more than there is: nothing is accepted of
    that request, and the same tree again goes on from the same keys."""
    from warp_b200 import ops
    ops.attn_status()
    a, b = tokens(3, 2 * PAGE + 3), tokens(4, 2 * PAGE - 2)
    lens = [len(a), len(b)]
    whole, d = decoder(model, 2, 2 * WIDE), decoder(model, 2, 5)
    first = whole.extend(torch.cat((a, b)), starts(lens), max(lens))
    assert torch.equal(d.extend(torch.cat((a, b)), starts(lens), max(lens)), first)
    ops.attn_status()
    assert d.pool[0] == 0
    trees = [tree_of(first[0], [1, 2, 3]), tree_of(first[1], [4, 5, 6])]
    both = (torch.cat(trees), i32(2 * UP), starts([4, 4]), 4)
    count, chosen = whole.verify(*both)
    ops.attn_status()
    tried, picked = d.verify(*both)
    starved()
    assert tried.tolist() == [count[0].item(), 0]
    assert picked.tolist() == [chosen[0].tolist(), [-1] * 4]
    assert d.kv_len.tolist() == [whole.kv_len[0].item(), len(b)]
    # once more with the same pages, and then with those of the first request
    again = (trees[1], i32(UP), starts([0, 4]), 4)
    tried, _ = d.verify(*again)
    starved()
    assert tried.tolist() == [0, 0] and d.kv_len[1] == len(b)
    d.kv_len[0] = 0
    fresh = decoder(model, 2, 2 * WIDE)
    fresh.extend(torch.cat((a, b)), starts(lens), max(lens))
    fresh.kv_len[0] = 0
    for _ in range(6):
        (n, picked), (m, want) = d.verify(*again), fresh.verify(*again)
        ops.attn_status()
        assert n.tolist() == m.tolist() and n[1] >= 1 and torch.equal(picked, want)
        assert torch.equal(d.kv_len, fresh.kv_len)
        last = picked[1, n[1] - 1]
        again = (tree_of(last, [7, (last.item() + 1) % V, 9]), i32(UP), starts([0, 4]), 4)


def test_a_prompt_past_its_row_of_pages_waits(model):  # noqa: F811
    """The same where the pool has pages and the request's row has no more entries."""
    from warp_b200 import ffi, ops
    ops.attn_status()
    d = decoder(model, 2, 3 * WIDE)
    long, short = tokens(5, WIDE * PAGE + 1), tokens(6, 9)
    got = d.extend(torch.cat((long, short)), starts([len(long), 9]), len(long))
    with pytest.raises(ffi.WarpError, match="length"):
        ops.attn_status()
    assert got[0] == -1 and got[1] >= 0
    assert d.kv_len.tolist() == [0, 9]


def test_a_captured_step_waits_for_pages(model):  # noqa: F811
    """Replays of one graph: a request that starves goes on when another has ended."""
    from warp_b200 import ops
    ops.attn_status()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        d = decoder(model, 2, 5)
        lens = [2 * PAGE + 3, 2 * PAGE - 2]
        first = d.extend(torch.cat((tokens(3, lens[0]), tokens(4, lens[1]))), starts(lens), max(lens))
        drafted = torch.full((8,), 5, dtype=torch.int32, device="cuda")
        drafted[0::4] = first
        parents, q_start = i32(2 * UP), starts([4, 4])
        kept = [x.clone() for x in (d.kv_len, d.held, d.pages, d.pool)]
        d.verify(drafted, parents, q_start, 4)      # the trunk wants a call before a capture
        starved()
        for x, y in zip((d.kv_len, d.held, d.pages, d.pool), kept):
            x.copy_(y)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            count, chosen = d.verify(drafted, parents, q_start, 4)
        graph.replay()
        assert count[0] >= 1 and count[1] == 0 and d.kv_len[1] == lens[1]
        starved()
        q_start.copy_(starts([0, 4]))
        drafted[:4] = drafted[4:].clone()
        d.kv_len[0] = 0
        graph.replay()
        ops.attn_status()
        assert count[0] == 0 and count[1] >= 1
        assert d.kv_len.tolist() == [0, lens[1] + count[1].item()]
