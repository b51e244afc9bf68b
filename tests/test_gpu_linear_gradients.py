"""Gradients of 16-bit layers behind sigmoid, gelu and silu carry one rounding, their own: dz enters both products as two
rounded parts, whatever the sizes.

Tolerance, per element: what two parts of a value leave of it is half a step of half a step, u^2 (u = eps / 2; below the
normal range half the smallest subnormal, `tiny`), the slope's product half a float32 step; a float32 sum of n products is
off by (n + 8) 2^-24 of their magnitudes twice over, and here every product comes in two parts, so (4 n + 16) 2^-24; then the
result's own half step.  With one part the first term is u, which is more than the whole of the rest."""
import ctypes

import pytest
import torch

from cafe_amd import _lib
from cafe_amd.linear import Slope, linear_backward

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24


def check(got, want, tol, what):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {off[bad].max():.3e} over {tol.expand_as(want)[bad].min():.3e}"


def rounded_once(m, k, n, t, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)                          # noqa: E731
    x, w, dy = r(m, k).to(t), (r(n, k) / k ** 0.5).to(t), r(m, n).to(t)
    s = torch.rand(m, n, device="cuda", generator=g) + 0.5
    u, tiny = torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps
    dx, dw, db = linear_backward(dy, x, w, Slope(s), "silu")
    dz, xd, wd = dy.double() * s.double(), x.double(), w.double()
    h = u * u * 1.02 + U32
    for got, want, mag, other, terms, what in (
            (dx, dz @ wd, dz.abs() @ wd.abs(), torch.ones_like(dz) @ wd.abs(), n, "dx"),
            (dw, dz.t() @ xd, dz.t().abs() @ xd.abs(), torch.ones_like(dz).t() @ xd.abs(), m, "dw"),
            (db[:, None], dz.sum(0)[:, None], dz.abs().sum(0)[:, None], torch.zeros(n, 1, device="cuda"), m, "db")):
        check(got, want, (h + (4 * terms + 16) * U32) * mag + tiny * other + 1.01 * u * want.abs() + tiny, what)
    return dx, dw, dz, xd, wd


TYPES = [torch.bfloat16, torch.float16]


# both sides of 4096 values, of 2^19 results and of 2^22 values of an operand; ragged and whole tiles; a long reduction
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (64, 64, 64), (65, 64, 64), (128, 367, 367), (300, 257, 130), (1030, 513, 700), (2048, 512, 384),
                                   (16384, 256, 1), (16385, 256, 1), (32768, 512, 4), (5000, 33, 40)])
def test_rounded_once(m, k, n, t):
    rounded_once(m, k, n, t, seed=m + n)


@pytest.mark.parametrize("t", TYPES)
def test_as_close_as_the_rounded_exact_gradients(t):
    """The distance from float64, as a norm, is that of the rounded float64 gradients (with dz in one part 1.4 times it); the
    float32 sums of at most 4096 terms add (2^-24 sqrt(4096)) at most, a hundredth of u."""
    dx, dw, dz, xd, wd = rounded_once(4096, 367, 256, t, seed=7)
    for got, want in ((dx, dz @ wd), (dw, dz.t() @ xd)):
        assert (got.double() - want).norm() <= 1.02 * (want.to(t).double() - want).norm()


def test_parts_behind_32_bits():
    """More than 2^32 values of dz: the second part starts behind them, and the last rows are theirs."""
    t, m, k, n = torch.bfloat16, (1 << 20) + 3, 8, 4104
    g = torch.Generator(device="cuda").manual_seed(1)
    dy = torch.empty(m, n, dtype=t, device="cuda")
    slopes = torch.empty(m, n, device="cuda")
    for at in range(0, m, 1 << 17):
        rows = min(1 << 17, m - at)
        dy[at:at + rows] = torch.randn(rows, n, device="cuda", generator=g)
        slopes[at:at + rows] = torch.rand(rows, n, device="cuda", generator=g) + 0.5
    x, w = (torch.randn(s, k, device="cuda", generator=g).to(t) for s in (m, n))
    dx, dw, db = linear_backward(dy, x, w, Slope(slopes), "silu")
    u, tiny = torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps
    for at in (0, m // 2, m - 300):
        dz = dy[at:at + 300].double() * slopes[at:at + 300].double()
        want, mag = dz @ w.double(), dz.abs() @ w.double().abs()
        check(dx[at:at + 300], want, (u * u * 1.02 + (4 * n + 17) * U32) * mag + 1.01 * u * want.abs() + tiny, "dx")
    out = (ctypes.c_int * 4)()
    _lib.check(_lib.load().cafe_linear_plan(m, k, n, 1, 4, 2, out), "cafe_linear_plan")
    row = -(-m // out[2]) + out[2]                              # additions in a row: a slice's and the slices'; db's, fewer than 2^12
    for c in (0, n // 2, n - 1):
        dz = dy[:, c].double() * slopes[:, c].double()
        want, mag = dz @ x.double(), dz.abs() @ x.double().abs()
        check(dw[c], want, (u * u * 1.02 + (4 * row + 17) * U32) * mag + 1.01 * u * want.abs() + tiny, "dw")
        check(db[c:c + 1], dz.sum()[None], 2 ** 12 * U32 * dz.abs().sum()[None] + 1.01 * u * dz.sum().abs()[None], "db")
    del dy, slopes, x, dx
    torch.cuda.empty_cache()
