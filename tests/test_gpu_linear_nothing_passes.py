"""A gradient that is not finite does not pass where the activation's slope is 0, whether the backward has the slopes or the
values before the activation; where the slope is not 0 it does."""
import math

import pytest
import torch

from cafe_amd.linear import Slope, linear_backward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["relu", "sigmoid", "gelu", "silu"])
def test_infinite_gradients(act, t):
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(s, device="cuda", generator=g).to(t)                    # noqa: E731
    m, k, n = 70, 45, 33
    x, w, z, dy = r(m, k), r(n, k), r(m, n), r(m, n)
    far = [-6e4, -math.inf] + ([6e4, math.inf] if act == "sigmoid" else [])             # slopes of 0
    for i, v in enumerate(far):
        for j, bad in enumerate((math.inf, -math.inf, math.nan)):
            z[10 + i, j], dy[10 + i, j] = v, bad
    slopes = torch.ones(m, n, device="cuda")
    slopes[10:10 + len(far), :3] = 0.0
    for kept in (z, Slope(slopes)):
        assert all(d.isfinite().all() for d in linear_backward(dy, x, w, kept, act))
    z[5, 7], dy[5, 7] = 1.0, math.inf                           # it is its row's and its column's
    dx, dw, db = linear_backward(dy, x, w, z, act)
    ok = torch.ones(m, dtype=torch.bool, device="cuda")
    ok[5] = False
    assert not dx[5].isfinite().any() and dx[ok].isfinite().all() and db[7] == math.inf
    assert not dw[7].isfinite().any() and torch.cat([dw[:7], dw[8:]]).isfinite().all()
