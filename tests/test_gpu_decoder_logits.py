"""Logits of steps of drafted trees against those of decoding token by token, at every node
that stands on the true path and in every step, however near the two best tokens are.

Both sides round, in other places: a step's normed states, queries, keys, values, softmax
weights and attention results to bf16 (u = 2^-8 relative, half a step), some six of a layer,
and the head's operand.  Over two layers and both sides these are 2 * (2 * 6 + 1) = 26, each
of a mean square of (u / sqrt 3)^2 of its norm at most and independent of the others:
sqrt(26 / 3) u = 0.0115 in all.  A single key of 37 in another's place moves a row by 0.056 and
more.  An expert that comes into the choice in another's place moves a row, too; nine of ten rows
are asked for."""
import pytest
import torch

from test_gpu_decoder import V, WIDE, decoder, i32, model, starts  # noqa: F401

pytestmark = pytest.mark.gpu

TOL = (26 / 3) ** 0.5 * 2.0 ** -8
STEPS = 14


def one_by_one(model, prompt):  # noqa: F811
    """Greedy tokens, and the logits that each was picked from."""
    d = decoder(model, 1, WIDE)
    heard, inner = [], d._logits

    def logits(h):
        heard.append(inner(h))
        return heard[-1]
    d._logits = logits
    tokens = [int(d.extend(i32(prompt), starts([len(prompt)]), len(prompt)))]
    while len(tokens) < STEPS:
        tokens.append(int(d.extend(i32(tokens[-1:]), starts([1]), 1)))
    return tokens, torch.cat([x[-1:] for x in heard])


@pytest.mark.parametrize("right", [3, 2, 1, 0])
def test_logits_of_drafted_trees(model, right):  # noqa: F811
    """The first `right` of three drafted tokens are the true ones, those behind them are not;
    node 0 is the true token whatever was picked."""
    from warp_b200 import ops
    g = torch.Generator().manual_seed(12)
    prompts = [torch.randint(0, V, (n,), generator=g).tolist() for n in (37, 5, 16)]
    true = [one_by_one(model, p) for p in prompts]
    d = decoder(model, 3, 3 * WIDE - 4)
    lens = [len(p) for p in prompts]
    d.extend(i32(sum(prompts, [])), starts(lens), max(lens))
    heard, inner = [], d._logits

    def logits(h):
        heard.append(inner(h))
        return heard[-1]
    d._logits = logits
    at, errors, steps = [1, 1, 1], [], 0
    while max(at) <= STEPS - 4:
        drafted, sizes = [], []
        for b, (tokens, _) in enumerate(true):
            after = tokens[at[b]:at[b] + 3]
            after = after[:right] + [(t + 1) % V for t in after[right:]]
            drafted += [tokens[at[b] - 1], (after[0] + 7) % V, after[0], (after[1] + 5) % V,
                        after[1], after[2], 3]
            sizes.append(7)
        count, chosen = d.verify(i32(drafted), i32([-1, 0, 0, 1, 2, 4, 4] * 3), starts(sizes), 7)
        steps += 1
        for b, (tokens, want) in enumerate(true):
            for k, node in enumerate([0, 2, 4, 5][:right + 1]):
                row, got = want[at[b] + k], heard[-1][7 * b + node]
                errors.append(float((got - row).norm() / row.norm()))
            c = int(count[b])
            # what is in the cache now is the true path
            assert 1 <= c <= right + 1 and chosen[b, :c - 1].tolist() == tokens[at[b]:at[b] + c - 1]
            at[b] += c
    ops.attn_status()
    assert d.kv_len.tolist() == [n + k - 1 for n, k in zip(lens, at)]
    # not by single tokens alone where more are right, so that moved keys are read
    assert steps == STEPS - 4 if right == 0 else steps < STEPS - 4
    assert len(errors) == 3 * steps * (right + 1)
    errors.sort()
    assert errors[len(errors) * 9 // 10] <= TOL, errors
