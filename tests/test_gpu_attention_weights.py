"""fp16 softmax weights far below a row's largest.

One key scores 17.5 above all others (in units of the exponential), its value
is 0 and the others' are 1000, so that the result is what the others weigh.
Tolerance: that of the attention tests, 2 (u |o| + (u + 2^-14) mag) with u = 2^-11,
and, for weights too small for a normal fp16 number where they are held against the
largest, n keys' absolute rounding of 2^-36 of the largest value each, doubled too.
"""
import pytest
import torch

from test_gpu_attention import Case

pytestmark = pytest.mark.gpu


def dominated(q, kv, at, value, prefix=0, D=64):
    c = Case(q, kv, 8, 2, D, 64, torch.float16, prefix=prefix, seed=33)
    c.q[:] = 1.0
    c.k[:], c.v[:] = 0.0, 1000.0
    for b in range(len(kv)):
        slot = c.pages[b][at // 64].long(), at % 64
        # 17.5 sqrt(D) / D: 2.1875 at D = 64, 1.546875 at 128 (17.501)
        c.k[slot] = 2.1875 if D == 64 else 1.546875
        c.v[slot] = value
    return c


def check(c, **kw):
    got = c.run(**kw)
    o, mag = c.want(causal=kw.get("causal", True))
    small = (max(c.kv_lens) + c.prefix) * 2.0 ** -36 * c.v.abs().nan_to_num().max().item()
    tol = 2 * (2.0 ** -11 * o.abs() + (2.0 ** -11 + 2.0 ** -14) * mag + small)
    err = (got.double() - o).abs()
    assert (err <= tol).all(), (err.max().item(), o.max().item(), tol.max().item())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("at", [0, 37])
def test_dominant_key_few_rows(cuda, D, at):
    check(dominated([1], [64], at, 0.0, D=D))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("at", [5, 4000])
def test_dominant_key_many_rows(cuda, D, at):
    check(dominated([40], [8192], at, 0.0, D=D), causal=False)


@pytest.mark.parametrize("q, kv", [([1, 1], [70, 300]), ([40, 30], [90, 200])])
def test_dominant_key_behind_a_prefix(cuda, q, kv):
    """The prefix's weights and the own keys' are held against different maxima."""
    check(dominated(q, kv, 30, 0.0, prefix=700), causal=False)


def test_rising_scores_fp16(cuda):
    """Each key outdoes those before it, so that the running maximum always moves."""
    for q, kv in (([1], [900]), ([140], [700])):
        c = Case(q, kv, 4, 1, 128, 64, torch.float16, seed=14)
        j = torch.arange(kv[0])
        c.q[:] = 1.0
        c.k[c.pages[0][j // 64].long(), j % 64] = (j * 0.02)[:, None, None].half()
        c.check()


@pytest.mark.parametrize("q, kv", [([1, 1, 3], [900, 77, 40]), ([170], [333])])
@pytest.mark.parametrize("sharp", [1.0, 8.0])
def test_largest_values_fp16(cuda, sharp, q, kv):
    """Weights above 1 of values near 65504: sums stay finite, small weights count."""
    c = Case(q, kv, 8, 2, 128, 32, torch.float16, seed=34, sharp=sharp)
    big = torch.rand(c.v.shape, generator=torch.Generator().manual_seed(35)) < 0.1
    c.v = torch.where(big & c.v.isfinite(), torch.full_like(c.v, 60000.0), c.v)
    check(c)
