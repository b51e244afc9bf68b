"""Activations and slopes of float32 layers over the whole line, value by value: K = 1 and weights of 1 hand z through.

Bounds.  e^-x is good to 3 half steps (the hardware's 2^x one step, the correction's sum half a one), the reciprocal to 2
after its Newton step, 1 + e to 1: sigmoid 8 2^-24 with its product, silu and the slopes' factors the same again.  gelu's
polynomial is evaluated to some 8 half steps and its fit is 1 off: with e (5), t (3) and the products 2^-20.  A slope that is a
sum is held against the magnitudes of its parts.  All of it relative, while the smallest factor is in float32's normal range;
below, that factor is taken as 0: 2^-125 times what it is multiplied by."""
import math

import pytest
import torch

from cafe_amd.linear import linear_forward

pytestmark = pytest.mark.gpu
REL, FLOOR = 2.0 ** -20, 2.0 ** -125


def points():
    z = [torch.linspace(-110, 110, 44001), torch.linspace(-14, 14, 28001), torch.linspace(-1e-3, 1e-3, 2001)]
    for c in (0.0, 12.98, 13.2, 20.0, 87.3365, 88.0, 88.7228, 91.0, 103.97, 104.0, 150.0, 1e4, 3e38):
        near = torch.tensor([c * (1 + k * 2.0 ** -23) for k in range(-8, 9)])
        z += [near, -near]
    z.append(torch.tensor([2.0 ** -k for k in range(1, 126)]))
    return torch.cat(z).cuda()


@pytest.mark.parametrize("n", [1, 128])                         # without LDS; through tiles
@pytest.mark.parametrize("act", ["sigmoid", "gelu", "silu"])
def test_over_the_line(act, n):
    x = points()
    z = x.double()
    one = torch.ones(n, 1, device="cuda")
    res = torch.zeros(len(x), n, device="cuda")                 # added as it is
    y, kept = linear_forward(x[:, None], one, None, act, res)
    s, t = torch.sigmoid(z), torch.sigmoid(-z)
    phi, d = 0.5 * torch.erfc(-z / math.sqrt(2)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "sigmoid":
        value, bound, slope, parts = s, REL / 2 * s, s * t, s * t
    elif act == "silu":
        value, bound, slope, parts = z * s, REL * (z * s).abs(), s + z * s * t, s + (z * s * t).abs()
    else:
        value, bound, slope, parts = z * phi, REL * (z * phi).abs(), phi + z * d, phi + (z * d).abs()
    floor = FLOOR * (1 + z.abs())
    for got, want, tol in ((y, value, bound + floor), (kept.values, slope, REL * parts + floor)):
        assert got.isfinite().all()
        for col in {0, n - 1}:
            off = (got[:, col].double() - want).abs()
            bad = off > tol
            assert not bad.any(), (act, float(z[bad][0]), float(got[:, col][bad][0]), float(want[bad][0]), float((off / want.abs())[bad].max()))
