"""cafe_amd.interact on the GPU against the formula in float64, pair by pair.

Tolerances: a float32 sum of n products is off by at most (2 n + 16) 2^-24 times the sum of their magnitudes (the matrix
units may order and align partial products in their own way); rounding to a type is half a step, eps / 2 relative, plus
half the smallest subnormal."""
import gc

import pytest
import torch

from cafe_amd.interact import dot_interaction

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
TYPES = [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.float32, torch.float16),
         (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)]


def rounding(want, t):
    return torch.finfo(t).eps / 2 * 1.01 * want.abs() + torch.finfo(t).smallest_normal * torch.finfo(t).eps


def make(f, b, d, te, t, dense, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    emb = torch.randn(f, b, d, device="cuda", generator=g).to(te)
    return (torch.randn(b, d, device="cuda", generator=g).to(t) if dense else None), emb, g


def rows_of(x, emb):
    r = emb.double().transpose(0, 1)
    return r if x is None else torch.cat([x.double()[:, None], r], 1)


def pairs_of(nf, itself):
    return [(i, j) for i in range(nf) for j in range(i + int(itself))]


def check(got, want, tol, what):
    assert got.shape == want.shape, what
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {(got.double() - want).abs()[bad].max():.3e}"


def verify(x, emb, itself, t, g):
    xl = None if x is None else x.detach().requires_grad_()
    el = emb.detach().requires_grad_()
    out = dot_interaction(xl, el, itself, dtype=t)
    r = rows_of(x, emb)
    nf, d = r.shape[1], r.shape[2]
    pairs = pairs_of(nf, itself)
    lead = 0 if x is None else d
    assert out.shape == (emb.shape[1], lead + len(pairs)) and out.dtype == t
    if lead:
        assert torch.equal(out[:, :lead], x)
    i = torch.tensor([p[0] for p in pairs], dtype=torch.long, device="cuda")
    j = torch.tensor([p[1] for p in pairs], dtype=torch.long, device="cuda")
    want = (r[:, i] * r[:, j]).sum(2)
    mag = (r[:, i].abs() * r[:, j].abs()).sum(2)
    check(out[:, lead:], want, (2 * d + 16) * U32 * mag + rounding(want, t), "out")
    assert torch.equal(dot_interaction(x, emb, itself, dtype=t), out)                # no autograd: the same
    if out.numel() == 0:
        return
    dout = torch.randn(out.shape, device="cuda", generator=g).to(t)
    grads = torch.autograd.grad(out, [el] if x is None else [el, xl], dout)
    dz = dout.double()[:, lead:]
    dr, dm = torch.zeros_like(r), torch.zeros_like(r)
    for k, (a, b) in enumerate(pairs):
        z = dz[:, k:k + 1]
        dr[:, a] += z * r[:, b]; dr[:, b] += z * r[:, a]
        dm[:, a] += (z * r[:, b]).abs(); dm[:, b] += (z * r[:, a]).abs()
    if lead:
        dr[:, 0] += dout.double()[:, :lead]; dm[:, 0] += dout.double()[:, :lead].abs()
    err = (2 * nf + 16) * U32 * dm
    k = int(bool(lead))
    check(grads[0], dr[:, k:].transpose(0, 1), (err[:, k:].transpose(0, 1) + rounding(dr[:, k:].transpose(0, 1), emb.dtype)), "demb")
    if lead:
        check(grads[1], dr[:, 0], err[:, 0] + rounding(dr[:, 0], t), "dx")


SIZES = [(1, 1, 1), (2, 3, 5), (7, 5, 16), (15, 9, 13), (16, 4, 64), (17, 6, 65), (22, 33, 16), (26, 70, 128), (31, 3, 7), (32, 5, 20),
         (40, 9, 200), (63, 3, 34), (64, 2, 16), (100, 2, 9), (127, 2, 130)]


@pytest.mark.parametrize("te,t", TYPES)
@pytest.mark.parametrize("f,b,d", SIZES)
def test_forward_and_backward(f, b, d, te, t):
    for dense, itself in ((True, False), (True, True), (False, False), (False, True)):
        if f + dense > 128:
            continue
        x, emb, g = make(f, b, d, te, t, dense, seed=f)
        verify(x, emb, itself, t, g)


def test_all_128_rows():
    x, emb, g = make(128, 3, 8, torch.float32, torch.float32, False)
    verify(None, emb, True, torch.float32, g)
    x, emb, g = make(0, 3, 8, torch.float32, torch.float32, True)                    # the dense row alone
    verify(x, emb, True, torch.float32, g)
    verify(x, emb, False, torch.float32, g)


@pytest.mark.parametrize("te,t", TYPES)
def test_strides(te, t):
    """Fields taken out of a larger array, rows at odd elements, [B, F, D] memory, a broadcast gradient."""
    g = torch.Generator(device="cuda").manual_seed(0)
    big = torch.randn(9, 20, 40, device="cuda", generator=g).to(te)
    emb = big[1:8:2, 3:17, 5:24]
    x = torch.randn(14, 21, device="cuda", generator=g).to(t)[:, 1:20]
    verify(x, emb, False, t, g)
    verify(x, torch.randn(14, 6, 19, device="cuda", generator=g).to(te).transpose(0, 1), True, t, g)
    verify(x, torch.randn(6, 19, 14, device="cuda", generator=g).to(te).transpose(1, 2), False, t, g)
    xl, el = x.detach().requires_grad_(), emb.detach().requires_grad_()
    a = torch.autograd.grad(dot_interaction(xl, el, dtype=t).sum(), [xl, el])
    out = dot_interaction(xl, el, dtype=t)
    assert all(torch.equal(p, q) for p, q in zip(a, torch.autograd.grad(out, [xl, el], torch.ones_like(out))))


def test_empty_batch_and_width():
    x, emb, g = make(5, 0, 8, torch.float32, torch.float32, True)
    xl, el = x.requires_grad_(), emb.requires_grad_()
    out = dot_interaction(xl, el)
    assert out.shape == (0, 8 + 15)
    dx, de = torch.autograd.grad(out, [xl, el], torch.zeros_like(out))
    assert dx.shape == (0, 8) and de.shape == (5, 0, 8)
    z = dot_interaction(torch.zeros(3, 0, device="cuda"), torch.zeros(2, 3, 0, device="cuda"))
    assert z.shape == (3, 3) and not z.any()
    z = dot_interaction(torch.zeros(0, 4, device="cuda"), torch.zeros(0, 0, 4, device="cuda"))
    assert z.shape == (0, 4)


def test_one_side_declined():
    x, emb, g = make(6, 11, 12, torch.float32, torch.float32, True)
    xl, el = x.detach().requires_grad_(), emb.detach().requires_grad_()
    out = dot_interaction(xl, el)
    dout = torch.randn(out.shape, device="cuda", generator=g)
    dx, de = torch.autograd.grad(out, [xl, el], dout)
    assert torch.equal(torch.autograd.grad(dot_interaction(xl, emb), xl, dout)[0], dx)
    assert torch.equal(torch.autograd.grad(dot_interaction(x, el), el, dout)[0], de)


def test_gradients_against_differences():
    """The form is a quadratic plus a linear one: central differences of the float64 formula are exact up to rounding."""
    x, emb, g = make(9, 6, 11, torch.float32, torch.float32, True)
    xl, el = x.detach().requires_grad_(), emb.detach().requires_grad_()
    out = dot_interaction(xl, el, True)
    dout = torch.randn(out.shape, device="cuda", generator=g)
    dx, de = torch.autograd.grad(out, [xl, el], dout)
    vx, ve = torch.randn(x.shape, device="cuda", generator=g).double(), torch.randn(emb.shape, device="cuda", generator=g).double()
    i, j = zip(*pairs_of(10, True))

    def f(h):
        r = rows_of(x.double() + h * vx, emb.double() + h * ve)
        return (dout.double() * torch.cat([r[:, 0], (r[:, list(i)] * r[:, list(j)]).sum(2)], 1)).sum()
    num = (f(0.5) - f(-0.5))
    mine = (dx.double() * vx).sum() + (de.double() * ve).sum()
    mag = (dx.double() * vx).abs().sum() + (de.double() * ve).abs().sum()
    assert abs(float(num - mine)) <= 1e-5 * float(mag)


def test_infinities_and_nan_stay_in_their_sample():
    x, emb, g = make(20, 9, 24, torch.float32, torch.float32, True)
    good = dot_interaction(x, emb)
    bad = emb.clone()
    bad[3, 4, 7], bad[19, 6, 0] = float("nan"), float("inf")
    out = dot_interaction(x, bad)
    ok = torch.ones(9, dtype=torch.bool, device="cuda")
    ok[4] = ok[6] = False
    assert torch.equal(out[ok], good[ok])
    pairs = pairs_of(21, False)
    with_row = torch.tensor([4 in p for p in pairs], device="cuda")                  # field 3 is row 4
    assert out[4, 24:][with_row].isnan().all() and torch.equal(out[4, 24:][~with_row], good[4, 24:][~with_row])


def test_graph_and_streams():
    x, emb, g = make(26, 300, 16, torch.float32, torch.bfloat16, True)
    xl, el = x.detach().requires_grad_(), emb.detach().requires_grad_()
    dout = torch.randn(300, 16 + 351, device="cuda", generator=g).bfloat16()

    def step():
        out = dot_interaction(xl, el, dtype=torch.bfloat16)
        return (out,) + torch.autograd.grad(out, [xl, el], dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    gc.collect()                     # a collected model frees device memory, which a capture forbids
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for s in range(3):
        with torch.no_grad():
            el.copy_(torch.randn(el.shape, device="cuda", generator=g))
            dout.copy_(torch.randn(dout.shape, device="cuda", generator=g))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        with torch.cuda.stream(side):
            other = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(other, want))


def test_a_batch_longer_than_a_launch():
    b = 2 ** 24 + 77
    g = torch.Generator(device="cuda").manual_seed(0)
    x, emb = torch.randn(b, 3, device="cuda", generator=g), torch.randn(1, b, 3, device="cuda", generator=g)
    xl, el = x.clone().requires_grad_(), emb.clone().requires_grad_()
    out = dot_interaction(xl, el)
    mag = (x.double().abs() * emb[0].double().abs()).sum(1)
    check(out[:, 3].detach(), (x.double() * emb[0].double()).sum(1), (2 * 3 + 16) * U32 * mag + U32 * mag, "out")
    dout = torch.randn(b, 4, device="cuda", generator=g)
    dx, de = torch.autograd.grad(out, [xl, el], dout)
    d = dout.double()
    want, size = d[:, :3] + d[:, 3:] * emb[0].double(), d[:, :3].abs() + (d[:, 3:] * emb[0].double()).abs()
    check(dx, want, (2 * 2 + 17) * U32 * size, "dx")
    want = d[:, 3:] * x.double()
    check(de[0], want, (2 * 2 + 17) * U32 * want.abs(), "demb")
    torch.cuda.empty_cache()


def test_offsets_past_32_bits():
    """Rows of the last field start behind 2^32 bytes and 2^31 elements."""
    f, b, d = 3, 700, 16
    g = torch.Generator(device="cuda").manual_seed(0)
    far = torch.empty(2 * (2 ** 30 + 2 ** 28) + b * d, device="cuda").as_strided((f, b, d), (2 ** 30 + 2 ** 28, d, 1))
    x, emb, _ = make(f, b, d, torch.float32, torch.float32, True)
    far.copy_(emb)
    a, z = (dot_interaction(x, e.detach().requires_grad_()) for e in (emb, far))
    assert torch.equal(a, z)
    verify(x, far, False, torch.float32, g)
    del far
    torch.cuda.empty_cache()


def test_wide_backward_in_a_graph():
    """90 rows: the backward's LDS passes 64 KB, which the kernel is told of under capture too."""
    x, emb, g = make(89, 40, 24, torch.float32, torch.float32, True)
    xl, el = x.detach().requires_grad_(), emb.detach().requires_grad_()
    dout = torch.randn(40, 24 + 90 * 89 // 2, device="cuda", generator=g)
    gc.collect()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(dot_interaction(xl, el), [xl, el], dout)
    for _ in range(3):
        with torch.no_grad():
            el.copy_(torch.randn(el.shape, device="cuda", generator=g))
        want = torch.autograd.grad(dot_interaction(xl, el), [xl, el], dout)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(got, want))
