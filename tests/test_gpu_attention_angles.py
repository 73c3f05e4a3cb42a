"""Rotation at far positions against exact angles.

The reduced angle is held as an fp32 fraction of a turn, off by 2^-26 at most,
which is 2 pi 2^-26 radians; sine and cosine are good to 2 units of 2^-24.  The angle
itself is to be exact: position times frequency, the frequency as it is given.
"""
import math
from decimal import Decimal, getcontext
from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu

PI = Fraction(Decimal("3.14159265358979323846264338327950288419716939937510582097494459"))
TOL = 2 * math.pi * 2.0 ** -26 + 2 * 2.0 ** -24


def exact(pos, f):
    a = pos * Fraction(f)
    return float(a - round(a / (2 * PI)) * 2 * PI)


@pytest.mark.parametrize("lo, hi", [(0, 5000), (10 ** 6, 2 ** 20 + 10 ** 6),
                                    (2 ** 31 - 1 - 10 ** 6, 2 ** 31 - 1), (-2 ** 31, -2 ** 31 + 999)])
def test_far_positions(cuda, lo, hi):
    from warp_b200 import ops
    g = torch.Generator().manual_seed(41)
    pos = torch.randint(lo, hi + 1, (48,), generator=g)
    f = torch.cat((torch.ones(1, dtype=torch.float64),
                   1 - 0.5 * torch.rand(31, generator=g, dtype=torch.float64)))
    x = torch.zeros(len(pos), 1, 64, device="cuda")
    x[..., :32] = 1.0                           # (1, 0) turns into (cos, sin)
    y, _ = ops.qk_norm_rope(x, None, pos.int().cuda(), f.cuda())
    a = torch.tensor([[exact(p, w) for w in f.tolist()] for p in pos.tolist()],
                     dtype=torch.float64)
    want = torch.cat((torch.cos(a), torch.sin(a)), 1)
    err = (y[:, 0].double().cpu() - want).abs().max().item()
    assert err <= TOL, err
