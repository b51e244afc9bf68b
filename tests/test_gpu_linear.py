"""cafe_amd.linear on the GPU against the formulas in float64.

Tolerances, derived per element.  A float32 sum of n products is off by at most n 2^-24 times the sum of their magnitudes
to first order; the matrix units may add partial products in an order (and with alignment) of their own, so 2 n + 16.  An
activation or its slope is evaluated in float32 to within 2^-20 absolute for unit arguments (a few ulp of exp and erfc);
gelu and silu have slopes below 1.2 and second derivatives below 1.  Rounding to the output type is half a step, eps / 2
relative, plus half the smallest subnormal."""
import gc

import pytest
import torch
import torch.nn as nn

from cafe_amd.linear import Slope, linear, linear_backward, linear_forward, run_mlp

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
ACTS = ["none", "relu", "sigmoid", "gelu", "silu"]
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps


def value(z, act):
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "sigmoid": lambda: torch.sigmoid(z),
            "gelu": lambda: z * 0.5 * torch.erfc(-z / 2 ** 0.5), "silu": lambda: z * torch.sigmoid(z)}[act]()


def slope(z, act):
    s = torch.sigmoid(z)
    return {"none": lambda: torch.ones_like(z), "relu": lambda: (z > 0).double(), "sigmoid": lambda: s * torch.sigmoid(-z),
            "gelu": lambda: 0.5 * torch.erfc(-z / 2 ** 0.5) + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5,
            "silu": lambda: s + z * s * torch.sigmoid(-z)}[act]()


def make(m, k, n, t, seed=0, bias=True, residual=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)                          # noqa: E731
    return (r(m, k).to(t), (r(n, k) / max(k, 1) ** 0.5).to(t), r(n).to(t) if bias else None, r(m, n).to(t) if residual else None,
            r(m, n).to(t))


def sum_error(a, b, n):
    """Bound of the float32 sum of n products a b^T."""
    return (2 * n + 16) * U32 * (a.abs() @ b.abs().t())


def check(got, want, tol, what):
    assert got.shape == want.shape, what
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {(got.double() - want).abs()[bad].max():.3e} over {tol.expand_as(want)[bad].min():.3e}"


def check_forward(y, kept, x, w, b, r, act):
    t, k = x.dtype, x.shape[1]
    xd, wd = x.double(), w.double()
    z = xd @ wd.t() + (b.double() if b is not None else 0)
    ez = sum_error(xd, wd, k) + 4 * U32 * z.abs()
    y0 = value(z, act) + (r.double() if r is not None else 0)
    check(y, y0, 1.2 * ez + 2 ** -20 * (1 + z.abs()) * (act not in ("none", "relu")) + 4 * U32 * y0.abs() + half_step(t) * 1.01 * y0.abs() + tiny(t), "y")
    if kept is not None and kept is not y:                      # act'(z); relu's: 0 or 1 by the sign, which z's error may turn
        k = kept.values if isinstance(kept, Slope) else kept
        s = slope(z, act)
        off = ez + 2 ** -20 * (1 + z.abs()) if act != "relu" else (z.abs() <= ez).double()
        assert k.dtype == torch.float32
        check(k, s, off + 2 * U32 * s.abs(), "kept")


def check_backward(grads, dy, x, w, kept, act):
    t, m, n = x.dtype, x.shape[0], w.shape[0]
    dyd, xd, wd = dy.double(), x.double(), w.double()
    given = isinstance(kept, Slope)
    s = kept.values.double() if given else slope(kept.double(), act) if act != "none" else torch.ones_like(dyd)
    dz = dyd * s
    # float32 value; slopes that come as they are cost the product's rounding alone
    ez = dyd.abs() * (0 if given or act in ("none", "relu") else 2 ** -20 * (1 + kept.double().abs())) + dz.abs() * 2 * U32
    rz = ez + (half_step(t) * 1.01 * dz.abs() + tiny(t) if act not in ("none", "relu") else 0)   # rounded before the products
    dx, dw, db = grads
    for got, want, err, what in (
            (dx, dz @ wd, rz @ wd.abs() + (2 * n + 16) * U32 * (dz.abs() @ wd.abs()), "dx"),
            (dw, dz.t() @ xd, rz.t() @ xd.abs() + (2 * m + 16) * U32 * (dz.t().abs() @ xd.abs()), "dw"),
            (db, dz.sum(0), ez.sum(0) + (2 * m + 16) * U32 * dz.abs().sum(0), "db")):
        if got is not None:
            check(got, want, err + half_step(t) * 1.01 * want.abs() + tiny(t), what)


SIZES = [(1, 1, 1), (1, 13, 16), (3, 5, 7), (2, 479, 1024), (5, 4100, 3), (63, 64, 65), (64, 32, 64), (65, 33, 16), (130, 479, 77),
         (257, 256, 1), (300, 8, 129), (128, 367, 367), (1000, 1, 300), (700, 130, 2), (1030, 257, 131)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_forward_and_backward(m, k, n, t):
    for i, act in enumerate(ACTS):
        x, w, b, r, dy = make(m, k, n, t, seed=m + i, bias=i != 1, residual=i % 2 == 0)
        y, kept = linear_forward(x, w, b, act, r)
        check_forward(y, kept, x, w, b, r, act)
        assert torch.equal(y, linear(x, w, b, act, r))
        check_backward(linear_backward(dy, x, w, kept, act), dy, x, w, kept, act)
        z = torch.randn(m, n, device="cuda").to(t)              # from the values before the activation
        check_backward(linear_backward(dy, x, w, z, act), dy, x, w, z, act)


@pytest.mark.parametrize("t", TYPES)
def test_large_enough_for_whole_tiles(t):
    x, w, b, r, dy = make(2048, 512, 384, t, residual=True)
    y, kept = linear_forward(x, w, b, "silu", r)
    check_forward(y, kept, x, w, b, r, "silu")
    check_backward(linear_backward(dy, x, w, kept, "silu"), dy, x, w, kept, "silu")


@pytest.mark.parametrize("t", TYPES)
def test_long_reduction_in_slices(t):
    """Few output tiles, a long sum: the reduction is split and joined, in forward and in both gradients."""
    for m, k, n in ((70, 5000, 40), (6000, 40, 30), (40, 30, 6000)):
        x, w, b, r, dy = make(m, k, n, t, residual=True)
        y, kept = linear_forward(x, w, b, "gelu", r)
        check_forward(y, kept, x, w, b, r, "gelu")
        a = linear_backward(dy, x, w, kept, "gelu")
        check_backward(a, dy, x, w, kept, "gelu")
        for p, q in zip(a, linear_backward(dy, x, w, kept, "gelu")):
            assert torch.equal(p, q)                            # fixed order of every sum


@pytest.mark.parametrize("t", TYPES)
def test_strided_and_unaligned_rows(t):
    """Views that start at odd elements, padded rows, a repeated row, a transposed weight, a broadcast residual."""
    m, k, n = 77, 61, 50
    g = torch.Generator(device="cuda").manual_seed(5)
    big = torch.randn(m + 2, k + 9, device="cuda", generator=g).to(t)
    x = big[1:m + 1, 3:3 + k]
    w = (torch.randn(k, n, device="cuda", generator=g) / 8).to(t).t()
    b = torch.randn(2 * n, device="cuda", generator=g).to(t)[::2]
    dy = torch.randn(m, n + 1, device="cuda", generator=g).to(t)[:, 1:]
    for act in ("none", "sigmoid"):
        y, kept = linear_forward(x, w, b, act)
        check_forward(y, kept, x, w, b, None, act)
        check_backward(linear_backward(dy, x, w, kept, act), dy, x, w, kept, act)
    one = x[:1].expand(m, k)                                    # row stride 0
    y, kept = linear_forward(one, w, b, "relu")
    check_forward(y, kept, one, w, b, None, "relu")
    check_backward(linear_backward(dy, one, w, kept, "relu"), dy, one, w, kept, "relu")
    r = torch.randn(m, 1, device="cuda", generator=g).to(t).requires_grad_()
    xl = x.detach().requires_grad_()
    y = linear(xl, w, b, "silu", r)
    check_forward(y.detach(), None, x, w, b, r.detach().expand(m, n), "silu")
    dr, = torch.autograd.grad(y, r, dy)
    check(dr, dy.double().sum(1, keepdim=True), (n * half_step(t) * dy.double().abs().sum(1, keepdim=True)) + tiny(t), "broadcast residual")


@pytest.mark.parametrize("t", TYPES)
def test_empty(t):
    x, w, b, r, dy = make(0, 5, 7, t)
    y, kept = linear_forward(x, w, b, "gelu")
    dx, dw, db = linear_backward(dy, x, w, kept, "gelu")
    assert y.shape == (0, 7) and dx.shape == (0, 5) and not dw.any() and not db.any() and dw.shape == (7, 5)
    x, w, b, r, dy = make(4, 0, 7, t, residual=True)
    y, kept = linear_forward(x, w, b, "relu", r)
    check_forward(y, kept, x, w, b, r, "relu")
    dx, dw, db = linear_backward(dy, x, w, kept, "relu")
    assert dx.shape == (4, 0) and dw.shape == (7, 0)
    check(db, (dy.double() * (kept.values > 0)).sum(0), 8 * half_step(t) * dy.double().abs().sum(0) + tiny(t), "db")
    x, w, b, r, dy = make(4, 6, 0, t)
    y, kept = linear_forward(x, w, b, "silu")
    dx, dw, db = linear_backward(dy, x, w, kept, "silu")
    assert y.shape == (4, 0) and dw.shape == (0, 6) and db.shape == (0,) and not dx.any() and dx.shape == (4, 6)


@pytest.mark.parametrize("t", TYPES)
def test_autograd_leading_dimensions_and_declined_gradients(t):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(3, 5, 19, device="cuda", generator=g).to(t).requires_grad_()
    w = (torch.randn(11, 19, device="cuda", generator=g) / 4).to(t).requires_grad_()
    b = torch.randn(11, device="cuda", generator=g).to(t).requires_grad_()
    r = torch.randn(5, 11, device="cuda", generator=g).to(t).requires_grad_()
    dy = torch.randn(3, 5, 11, device="cuda", generator=g).to(t)
    y = linear(x, w, b, "silu", r)
    dx, dw, db, dr = torch.autograd.grad(y, [x, w, b, r], dy)
    x2, kept = x.detach().view(15, 19), linear_forward(x.detach().view(15, 19), w.detach(), b.detach(), "silu")[1]
    check_backward((dx.view(15, 19), dw, db), dy.view(15, 11), x2, w.detach(), kept, "silu")
    check(dr, dy.double().sum(0), 3 * half_step(t) * dy.double().abs().sum(0) + tiny(t), "dr")
    one, = torch.autograd.grad(linear(x, w.detach(), b.detach(), "silu"), x, dy)
    assert torch.equal(one, dx)
    only, = torch.autograd.grad(linear(x.detach(), w.detach(), b, "relu"), b, dy)
    z = x.detach().double() @ w.detach().double().t() + b.detach().double()
    check(only, (dy.double() * (z > 0)).sum((0, 1)), 16 * half_step(t) * dy.double().abs().sum((0, 1)) + tiny(t), "db alone")
    v = linear(x.detach()[0, 0], w.detach(), b.detach(), "gelu")
    assert v.shape == (11,)
    with pytest.raises(RuntimeError):                           # differentiable once
        gx, = torch.autograd.grad(linear(x, w, b, "silu").sum(), x, create_graph=True)
        gx.sum().backward()


@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(act):
    """Directional derivatives of the float64 formula by central differences (error h^2 times the third derivative, below
    1e-6 of the sums here) against the inner products with the kernel's float32 gradients."""
    x, w, b, r, dy = make(37, 29, 23, torch.float32, seed=9)
    if act == "relu":                                           # the formula has a corner: keep the sums off it
        b = b + 10.0
    y, kept = linear_forward(x, w, b, act)
    dx, dw, db = linear_backward(dy, x, w, kept, act)
    g = torch.Generator(device="cuda").manual_seed(2)
    vx, vw, vb = (torch.randn(s.shape, device="cuda", generator=g).double() for s in (x, w, b))
    f = lambda h: (dy.double() * value((x.double() + h * vx) @ (w.double() + h * vw).t() + b.double() + h * vb, act)).sum()   # noqa: E731
    h = 1e-4
    num = (f(h) - f(-h)) / (2 * h)
    mine = (dx.double() * vx).sum() + (dw.double() * vw).sum() + (db.double() * vb).sum()
    scale = (dx.double() * vx).abs().sum() + (dw.double() * vw).abs().sum() + (db.double() * vb).abs().sum()
    assert abs(float(num - mine)) <= 1e-5 * float(scale)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_infinities_and_nan_stay_in_their_rows(t, act):
    """A row that holds NaN or infinities makes its own outputs what the formula makes them and leaves the others."""
    m, k, n = 70, 45, 33
    x, w, b, r, dy = make(m, k, n, t, seed=3)
    good, _ = linear_forward(x, w, b, act)
    x2 = x.clone()
    x2[5, 7], x2[66, 44] = float("nan"), float("inf")
    y, kept = linear_forward(x2, w, b, act)
    ok = torch.ones(m, dtype=torch.bool, device="cuda")
    ok[5] = ok[66] = False
    assert torch.equal(y[ok], good[ok])
    assert y[5].isnan().all()
    sign = w[:, 44] > 0
    limit = {"sigmoid": (1.0, 0.0), "relu": (float("inf"), 0.0), "gelu": (float("inf"), 0.0), "silu": (float("inf"), 0.0),
             "none": (float("inf"), float("-inf"))}[act]
    assert (y[66][sign] == limit[0]).all() and (y[66][~sign & (w[:, 44] < 0)] == limit[1]).all()
    kept2 = torch.randn(m, n, device="cuda").to(t)
    kept2[5, 3], kept2[6, 3] = float("inf"), float("-inf")
    dx, dw, db = linear_backward(dy, x, w, kept2, act)
    assert dx.isfinite().all() and dw.isfinite().all() and db.isfinite().all()
    if act == "relu":                                           # an infinite gradient where nothing passes does not
        kept2[9, 4], dy[9, 4] = -1.0, float("inf")
        kept2[10, 4], dy[10, 4] = 0.0, float("nan")
        for kept in (kept2, Slope((kept2 > 0).float())):
            dx, dw, db = linear_backward(dy, x, w, kept, act)
            assert dx.isfinite().all() and dw.isfinite().all() and db.isfinite().all()


@pytest.mark.parametrize("t", TYPES)
def test_graph_capture_and_replay(t):
    """Two captured steps that share inputs, replayed among eager work, give the eager results every time."""
    x, w, b, r, dy = make(200, 479, 64, t, residual=True)

    def step(act):
        y, kept = linear_forward(x, w, b, act, r)
        return (y,) + linear_backward(dy, x, w, kept, act)

    graphs = []
    for act in ("silu", "relu"):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(act)
        torch.cuda.current_stream().wait_stream(side)
        gc.collect()                     # a collected model frees device memory, which a capture forbids
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(act)
        graphs.append((g, out, act))
    for seed in range(3):
        nx, _, _, nr, ndy = make(200, 479, 64, t, seed=50 + seed, residual=True)
        x.copy_(nx); r.copy_(nr); dy.copy_(ndy)
        want = [step(act) for _, _, act in graphs]
        for g, _, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, out, _), ref in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, ref))


def test_two_streams_at_once():
    sets = [make(300, 700, 90, torch.float32, seed=s) for s in range(2)]
    want = [linear_backward(s[4], s[0], s[1], linear_forward(s[0], s[1], s[2], "gelu")[1], "gelu") for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for q, (s, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                got[q] = linear_backward(s[4], s[0], s[1], linear_forward(s[0], s[1], s[2], "gelu")[1], "gelu")
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_mlp_of_modules(t):
    """run_mlp over nn.Sequential is the layers' `linear` calls in order, the residual in the last one, and its
    parameters get their gradients."""
    torch.manual_seed(0)
    layers = nn.Sequential(nn.Linear(13, 40), nn.ReLU(), nn.Linear(40, 24), nn.SiLU(), nn.Linear(24, 9), nn.Linear(9, 1), nn.Sigmoid()).cuda().to(t)
    x = torch.randn(50, 13, device="cuda").to(t)
    wide = torch.randn(50, 1, device="cuda").to(t)
    out = run_mlp(layers, x, wide)
    params = list(layers.parameters())
    got = torch.autograd.grad(out, params, torch.ones_like(out))
    h, steps = x, []
    for i, act in ((0, "relu"), (2, "silu"), (4, "none"), (5, "sigmoid")):
        y, kept = linear_forward(h, layers[i].weight, layers[i].bias, act, wide if i == 5 else None)
        steps.append((h, layers[i].weight, kept, act))
        h = y
    assert torch.equal(h, out)
    d, want = torch.ones_like(out), []
    for h, w, kept, act in reversed(steps):
        d, dw, db = linear_backward(d, h, w, kept, act)
        want = [dw, db] + want
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_more_rows_than_a_grid_is_wide(t):
    """One output column: 16 rows per workgroup, 2^20 workgroups side by side, the rest in a second row of them."""
    m, k = 16 * 2 ** 20 + 50, 5
    x, w, b, _, _ = make(4, k, 1, t)
    x = torch.randn(m, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(t)
    y = linear(x, w, b)
    xd, wd = x.double(), w.double()
    want = xd @ wd.t() + b.double()
    check(y, want, sum_error(xd, wd, k) + 4 * U32 * want.abs() + half_step(t) * 1.01 * want.abs() + tiny(t), "y")
    torch.cuda.empty_cache()


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_offsets_past_32_bits(t):
    """Rows 2^24 elements apart: the last ones start behind 2^31 elements, in every operand of both passes."""
    m, k, n, far = 150, 130, 200, 2 ** 24
    x, w, b, _, dy = make(m, k, n, t)

    def spread(a):
        out = torch.empty((a.shape[0] - 1) * far + a.shape[1], dtype=t, device="cuda").as_strided(a.shape, (far, 1))
        out.copy_(a)
        return out
    near = linear_forward(x, w, b, "silu")
    want = linear_backward(dy, x, w, near[1], "silu")
    xs = spread(x)
    assert torch.equal(linear_forward(xs, w, b, "silu")[0], near[0])
    got = linear_backward(dy, xs, w, near[1], "silu")
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    del xs
    ws = spread(w)
    assert torch.equal(linear_forward(x, ws, b, "silu")[0], near[0])
    got = linear_backward(dy, x, ws, near[1], "silu")
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    del ws
    ds = spread(dy)
    got = linear_backward(ds, x, w, near[1], "silu")
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    del ds
    torch.cuda.empty_cache()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_the_bias_gradient_alone(t, act):
    """The same bits as beside the other gradients, for one product of slices and for a whole one."""
    for m, k, n in ((70, 30, 50), (5000, 20, 33), (3, 200, 600)):
        x, w, b, _, dy = make(m, k, n, t)
        kept = linear_forward(x, w, b, act)[1]
        want = linear_backward(dy, x, w, kept, act)
        db = linear_backward(dy, x, w, kept, act, need=(False, False, True))
        assert db[0] is None and db[1] is None and torch.equal(db[2], want[2])


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [(9689, 83, 5), (16, 300, 200), (1, 40, 3), (900, 7, 4)])
def test_few_results_are_rounded_once(m, k, n, t):
    """Where min(values of dz, results) is at most 4096, dz enters the products in two parts: what is left of its rounding
    is half a step of half a step, the rounding of the result stands alone."""
    x, w, _, _, dy = make(m, k, n, t)
    s = torch.rand(m, n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) + 0.5
    dx, dw, _ = linear_backward(dy, x, w, Slope(s), "silu")
    dz, xd, wd = dy.double() * s.double(), x.double(), w.double()
    h = half_step(t) ** 2 * 1.02 + U32                      # of a value of dz; below float16's normal range half a subnormal step
    low = tiny(t)
    for got, want, mag, other, terms in ((dx, dz @ wd, dz.abs() @ wd.abs(), torch.ones_like(dz) @ wd.abs(), n),
                                         (dw, dz.t() @ xd, dz.t().abs() @ xd.abs(), torch.ones_like(dz).t() @ xd.abs(), m)):
        if min(m * n, want.numel()) <= 4096:
            check(got, want, (h + (2 * 2 * terms + 16) * U32) * mag + low * other + half_step(t) * 1.01 * want.abs() + tiny(t), "product")
