"""cafe_amd.adamw on the GPU: moments and 8-bit codes against float32 operations in the stated order (equal bits), updated
parameters against the formula in float64.

Tolerance of a parameter: keep, step size, betas and eps are float32 numbers and the update is four float32 operations
with a square root and a division, each half a step: 16 2^-24 of the update's magnitude, 4 2^-24 of the parameter, then
half a step of the parameter's type."""
import gc
import math

import pytest
import torch

from cafe_amd.adamw import AdamW, Moment8, adamw_step, adamw_tick, moment8_values

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.02)
SIZES = [1, 2, 3, 5, 255, 256, 257, 1000, 4095, 4096, 4097, 70001]


def table(second):
    """Every value a code stands for at E = 0, in code order (float64), from the format's definition."""
    low = -30 if second else -14
    out = []
    for c in range(255 if second else 128):
        field, man = c >> 3, c & 7
        out.append(man * 2.0 ** (low - 3) if field == 0 else (8 + man) * 2.0 ** (field - 1 + low - 3))
    return torch.tensor(out, dtype=torch.float64)


def encode(x, second):
    """Nearest code by search in the table, ties to the even code."""
    x = x.detach().cpu().double().reshape(-1)
    t = table(second)
    codes, exps = [], []
    for k in range(0, x.numel(), 256):
        b = x[k:k + 256]
        fin = b[b.isfinite()].abs()
        top = float(fin.max()) if fin.numel() else 0.0
        e = max(math.frexp(top)[1] - 1, -126) if top > 0 else -126
        a = torch.where(b.isfinite(), b.abs(), torch.zeros_like(b)) * 2.0 ** -e
        hi = torch.searchsorted(t, a).clamp(max=t.numel() - 1)
        lo = (hi - 1).clamp(min=0)
        du, dl = (t[hi] - a).abs(), (a - t[lo]).abs()
        c = torch.where((dl < du) | ((dl == du) & (lo % 2 == 0)), lo, hi)
        if second:
            c = torch.where((c == 0) & (b > 0), torch.ones_like(c), c)
            c = torch.where(b.isfinite(), c, torch.full_like(c, 0xff))
        else:
            c = torch.where((b < 0) & (c > 0), c + 128, c)
            c = torch.where(b.isfinite(), c, torch.full_like(c, 0x80))
        codes.append(c)
        exps.append(e + 127)
    return torch.cat(codes).to(torch.uint8).cuda(), torch.tensor(exps, dtype=torch.uint8, device="cuda")


def decode(m8, second):
    """The values of codes, from the table."""
    t = table(second)
    c = m8.codes.cpu().long()
    v = t[(c if second else c & 127).clamp(max=t.numel() - 1)]
    if not second:
        v = torch.where(c >= 128, -v, v)
    e = (m8.exponents.cpu().long() - 127).repeat_interleave(256)[:c.numel()]
    v = v * torch.exp2(e.double())
    v[c == (0xff if second else 0x80)] = math.inf if second else math.nan
    return v.float().cuda()


def make(n, t, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda: torch.randn(n, device="cuda", generator=g)                             # noqa: E731
    spread = torch.exp(2 * r())
    return (r() * 0.1).to(t), (r() * spread * 1e-3).to(t), r() * spread * 3e-4, (r() * spread * 1e-3) ** 2


def reference(p, g, m, v, step):
    """float32 moments in the stated order, float64 parameter and its tolerance before the type's rounding."""
    b1, b2 = HYPER["betas"]
    g = g.float()
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    upd = HYPER["lr"] / (1 - b1 ** step) * m.double() / (v.double().sqrt() / math.sqrt(1 - b2 ** step) + HYPER["eps"])
    new = p.double() * (1 - HYPER["lr"] * HYPER["weight_decay"]) - upd
    return m, v, new, 16 * U32 * upd.abs() + 4 * U32 * p.double().abs() + 2 * U32 * new.abs()


def rounding(want, t):
    return torch.finfo(t).eps / 2 * 1.01 * want.abs() + torch.finfo(t).smallest_normal * torch.finfo(t).eps


def near(got, want, tol, what):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {(got.double() - want).abs()[bad].max():.3e}"


@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("t", TYPES)
def test_steps(t, bits, master):
    """Three steps over tensors of many sizes at once (more than one launch's worth of them)."""
    sets = [make(n, t, seed=i) for i, n in enumerate(SIZES * 5)]
    p, g, m, v = ([s[k].clone() for s in sets] for k in range(4))
    if bits == 8:
        m8, v8 = [Moment8(*encode(x, False)) for x in m], [Moment8(*encode(x, True)) for x in v]
        m, v = [decode(x, False) for x in m8], [decode(x, True) for x in v8]
    w = [x.float() for x in p] if master else None
    for step in (1, 2, 1000):
        g = [x * (1.5 - 0.5 * (step == 2)) for x in g]
        want = [reference(w[i] if master else p[i], g[i], m[i], v[i], step) for i in range(len(p))]
        adamw_step(p, g, m8 if bits == 8 else m, v8 if bits == 8 else v, step=step, masters=w, **HYPER)
        if bits == 8:
            got_m, got_v = moment8_values(m8, v8)
        for i, (rm, rv, new, tol) in enumerate(want):
            if bits == 8:
                cm, cv = Moment8(*encode(rm, False)), Moment8(*encode(rv, True))
                assert torch.equal(m8[i].exponents, cm.exponents) and torch.equal(v8[i].exponents, cv.exponents)
                assert torch.equal(m8[i].codes, cm.codes) and torch.equal(v8[i].codes, cv.codes)
                m[i], v[i] = decode(cm, False), decode(cv, True)
                assert torch.equal(got_m[i], m[i]) and torch.equal(got_v[i], v[i])
            else:
                assert torch.equal(m[i], rm) and torch.equal(v[i], rv)
            if master:
                near(w[i], new, tol, "master")
                assert torch.equal(p[i], w[i].to(t))
            else:
                near(p[i], new, tol + rounding(new, t), "p")


def test_codes_of_the_format():
    """Every code of every binade survives a step that changes nothing (g = 0, betas = 0 keep no history: m = v = 0), and
    values half way between codes, zeros, subnormals, the largest floats and what is not finite encode as defined."""
    x = torch.cat([table(True), (table(True)[1:] + table(True)[:-1]) / 2]).float().cuda()
    cases = [x, x * 2.0 ** -100, x * 2.0 ** 126, torch.zeros(300, device="cuda"),
             torch.tensor([1e-45, 1e-40, 0.0, 2.0 ** -126] * 70, device="cuda"),
             torch.tensor([3.4e38, 1.0, 0.0, math.inf, 1e-30, math.nan] * 50, device="cuda")]
    for c in cases:
        for sign in (1.0, -1.0):
            n = c.numel()
            p, m, v = torch.zeros(n, device="cuda"), Moment8.zeros(n, "cuda"), Moment8.zeros(n, "cuda")
            adamw_step([p], [c * sign], [m], [v], step=1, lr=0.0, betas=(0.0, 0.0), eps=1.0, weight_decay=0.0)
            g = c * sign
            em, ev = Moment8(*encode(g, False)), Moment8(*encode(g * g, True))
            assert torch.equal(m.codes, em.codes) and torch.equal(m.exponents, em.exponents)
            assert torch.equal(v.codes, ev.codes) and torch.equal(v.exponents, ev.exponents)
            gm, gv = moment8_values([m], [v])
            assert torch.equal(gm[0].nan_to_num(7.0), decode(em, False).nan_to_num(7.0)) and torch.equal(gv[0], decode(ev, True))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_gradient_that_is_not_finite_stays_with_its_value(bits):
    n = 1000
    p, g, m, v = make(n, torch.float32, 0)
    if bits == 8:
        m, v = Moment8(*encode(m, False)), Moment8(*encode(v, True))
    state = lambda: [p.clone()] + ([t.clone() for t in m + v] if bits == 8 else [m.clone(), v.clone()])   # noqa: E731
    keep = state()
    adamw_step([p], [g], [m], [v], step=5, **HYPER)
    good = state()
    p.copy_(keep[0])
    for dst, src in zip(m + v if bits == 8 else (m, v), keep[1:]):
        dst.copy_(src)
    g[300], g[700] = math.nan, math.inf
    adamw_step([p], [g], [m], [v], step=5, **HYPER)
    ok = torch.ones(n, dtype=torch.bool, device="cuda")
    ok[300] = ok[700] = False
    assert torch.equal(p[ok], good[0][ok]) and p[300].isnan()
    for a, b in zip(state()[1:], good[1:]):
        if a.numel() == n:
            assert torch.equal(a[ok], b[ok])
        else:                                                   # a block's exponent may fall where its largest value left
            assert (a <= b).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_unaligned_views(bits):
    """Parameters, gradients and moments that start at any element of their storage; neighbours stay as they were."""
    n, t = 777, torch.bfloat16
    p0, g0, m0, v0 = make(n, t, 4)
    if bits == 8:
        mc, vc = encode(m0, False), encode(v0, True)

    def put(x, off):
        buf = torch.full((x.numel() + 16,), 9, dtype=x.dtype, device="cuda")
        buf[off:off + x.numel()] = x.view(-1)
        return buf, buf[off:off + x.numel()]
    outs = []
    for off in (0, 1, 3, 7):
        pb, p = put(p0, off)
        gb, g = put(g0, off + 1)
        if bits == 8:
            bufs = [put(x, off + k) for k, x in enumerate(mc + vc)]
            m, v = Moment8(bufs[0][1], bufs[1][1]), Moment8(bufs[2][1], bufs[3][1])
        else:
            bufs = [put(m0, off), put(v0, off + 1)]
            m, v = bufs[0][1], bufs[1][1]
        adamw_step([p], [g], [m], [v], step=3, **HYPER)
        outs.append([p.clone()] + [x.clone() for _, x in bufs])
        for b, x in [(pb, p)] + bufs:
            start = x.storage_offset()
            assert (b[:start] == 9).all() and (b[start + x.numel():] == 9).all()
    for o in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(o, outs[0]))


def test_empty_and_strided_gradients():
    p, g, m, v = make(12, torch.float32, 0)
    p, m, v = p.view(3, 4), m.view(3, 4), v.view(3, 4)
    q, qm, qv = p.clone(), m.clone(), v.clone()
    z = [torch.zeros(0, device="cuda") for _ in range(4)]
    adamw_step([z[0], p], [z[1], g.view(4, 3).t()], [z[2], m], [z[3], v], step=1, **HYPER)
    adamw_step([q], [g.view(4, 3).t().contiguous()], [qm], [qv], step=1, **HYPER)
    assert torch.equal(p, q) and torch.equal(m, qm) and torch.equal(v, qv)
    adamw_step([z[0]], [z[1]], [Moment8.zeros(0, "cuda")], [Moment8.zeros(0, "cuda")], step=1, **HYPER)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("t", TYPES)
def test_optimizer_is_the_function(t, bits):
    """AdamW against adamw_step, over groups with their own numbers, a parameter that misses a step, and a checkpoint."""
    torch.manual_seed(0)
    shapes = [(5, 7), (300,), (1,), (64, 65)]
    ps = [torch.nn.Parameter(torch.randn(s, device="cuda").to(t)) for s in shapes]
    opt = AdamW([dict(params=ps[:2], lr=1e-2), dict(params=ps[2:], weight_decay=0.3, betas=(0.8, 0.9))], state_bits=bits)
    hyper = [dict(lr=1e-2, betas=(0.9, 0.999), weight_decay=0.01)] * 2 + [dict(lr=1e-3, betas=(0.8, 0.9), weight_decay=0.3)] * 2
    qs = [p.detach().clone() for p in ps]
    ws = [q.float() for q in qs] if t is not torch.float32 else None
    new = (lambda q: Moment8.zeros(q.numel(), "cuda")) if bits == 8 else (lambda q: torch.zeros(q.shape, device="cuda"))
    ms, vs, steps = [new(q) for q in qs], [new(q) for q in qs], [0] * 4
    for it in range(6):
        for i, p in enumerate(ps):
            p.grad = None if (i, it) == (1, 2) else torch.randn(p.shape, device="cuda").to(t)
        opt.step()
        for i, p in enumerate(ps):
            if p.grad is not None:
                steps[i] += 1
                adamw_step([qs[i]], [p.grad], [ms[i]], [vs[i]], step=steps[i], masters=None if ws is None else [ws[i]], **hyper[i])
            assert torch.equal(p.detach(), qs[i]), (it, i)
        if it == 3:                                             # through a checkpoint into a new optimizer
            import io
            f = io.BytesIO()
            torch.save(opt.state_dict(), f)
            f.seek(0)
            opt = AdamW([dict(params=ps[:2]), dict(params=ps[2:])], state_bits=bits)
            opt.load_state_dict(torch.load(f, weights_only=True))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step(bits):
    """capturable: replays advance the device's step count and read the learning rate there; every replay is the eager step."""
    t = torch.bfloat16
    p = torch.nn.Parameter(torch.randn(5000, device="cuda").to(t))
    q = torch.nn.Parameter(p.detach().clone())
    lr = torch.full((1,), 1e-2, device="cuda")
    opt = AdamW([p], lr=lr, state_bits=bits, capturable=True)
    ref = AdamW([q], lr=1e-2, state_bits=bits)
    grad = torch.randn(5000, device="cuda").to(t)
    p.grad, q.grad = grad, grad
    opt.step(); ref.step()
    assert torch.equal(p, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    ref.step()
    gc.collect()                     # a collected model frees device memory, which a capture forbids
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
        with pytest.raises(Exception, match="captured step"):
            adamw_step([q], [grad], [torch.zeros(5000, device="cuda")], [torch.zeros(5000, device="cuda")], step=1, lr=0.1)
    for k in range(4):
        grad.copy_(torch.randn(5000, device="cuda"))
        new = 1e-2 / (k + 1)
        lr.fill_(new)
        ref.param_groups[0]["lr"] = float(lr)
        graph.replay()
        ref.step()
        torch.cuda.synchronize()
        assert torch.equal(p, q), k
    assert opt.state_dict()["param_groups"][0]["device_step"] == {str(p.device): 6}


def test_two_streams_and_repeats():
    sets = [make(50001, torch.float32, s) for s in range(2)]
    outs = []
    for rep in range(2):
        cur = [[x.clone() for x in s] for s in sets]
        streams = [torch.cuda.Stream() for _ in cur]
        torch.cuda.synchronize()
        for step in range(1, 4):
            for (p, g, m, v), st in zip(cur, streams):
                with torch.cuda.stream(st):
                    adamw_step([p], [g], [m], [v], step=step, **HYPER)
        torch.cuda.synchronize()
        outs.append(cur)
    for a, b in zip(*outs):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_tick():
    step, factors = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(3, device="cuda")
    for t in (1, 2, 3):
        adamw_tick(step, factors, lr=0.01, betas=(0.9, 0.99), weight_decay=0.1)
        want = torch.tensor([0.01 / (1 - 0.9 ** t), 1 / math.sqrt(1 - 0.99 ** t), 1 - 0.01 * 0.1], dtype=torch.float64)
        # the double's powers are good to a few 2^-52, 1 - 0.99 loses two digits of that: float32's half step remains
        near(factors.cpu(), want, 1.01 * U32 * want, "factors")
        assert int(step) == t


def test_a_capture_creates_no_moments():
    """Zeros written in a capture would be written again by every replay."""
    p, late = (torch.nn.Parameter(torch.ones(10, device="cuda")) for _ in range(2))
    opt = AdamW([p, late], capturable=True)
    p.grad = torch.ones(10, device="cuda")
    opt.step()
    late.grad = torch.ones(10, device="cuda")
    gc.collect()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph), pytest.raises(Exception, match="before the capture"):
        opt.step()
    opt.step()                                                                       # eager: creates them
    assert len(opt.state[late]) > 1


def test_a_backward_notices_the_step():
    p = torch.nn.Parameter(torch.ones(4, device="cuda"))
    loss = (p * p).sum()
    adamw_step([p.detach()], [torch.ones(4, device="cuda")], [torch.zeros(4, device="cuda")], [torch.zeros(4, device="cuda")], step=1, lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("t,bits", [(torch.bfloat16, 8), (torch.float32, 32)])
def test_tensors_longer_than_a_launch(t, bits):
    """2^22 workgroups of 2048 (8 bits) or 1024 values and a few more: repeated rows get what one row gets, in every piece."""
    row, rows = 256 * 4097, 8200 if bits == 8 else 4100
    assert row * rows > 2 ** 22 * (2048 if bits == 8 else 1024)
    g = torch.Generator(device="cuda").manual_seed(0)
    small = [torch.randn(row, device="cuda", generator=g).to(t) for _ in range(2)]
    def spread(x):
        return x.repeat(rows)
    p, grad = (spread(x) for x in small)
    if bits == 8:
        ms, ml = ([Moment8.zeros(n, "cuda") for _ in range(2)] for n in (row, row * rows))
        ws, wl = [small[0].float()], [p.float()]
    else:
        ms, ml = ([torch.zeros(n, device="cuda") for _ in range(2)] for n in (row, row * rows))
        ws = wl = None
    for step in (1, 2):
        adamw_step([small[0]], [small[1]], [ms[0]], [ms[1]], step=step, masters=ws, **HYPER)
        adamw_step([p], [grad], [ml[0]], [ml[1]], step=step, masters=wl, **HYPER)

    def same(long, one):
        return all(torch.equal(r, one) for r in long.view(rows, -1))
    assert same(p, small[0])
    if bits == 8:
        assert same(wl[0], ws[0]) and all(same(a, b) for k in range(2) for a, b in zip(ml[k], ms[k]))
        del p, grad, wl
        (lm,), (lv,) = moment8_values([ml[0]], [ml[1]])
        (sm,), (sv,) = moment8_values([ms[0]], [ms[1]])
        assert same(lm, sm) and same(lv, sv)
    else:
        assert same(ml[0], ms[0]) and same(ml[1], ms[1])
    p = grad = wl = ml = lm = lv = None
    torch.cuda.empty_cache()


@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("t", TYPES)
def test_steps_past_the_caches(t, bits, master):
    """More than 480 MB in a call: the arrays go past the caches, from addresses off any 16-byte boundary too; repeated rows
    get what one row gets."""
    row, rows = 256 * 4097, 52
    g = torch.Generator(device="cuda").manual_seed(1)
    small = [torch.randn(row, device="cuda", generator=g).to(t) for _ in range(2)]

    def spread(x):
        out = torch.empty(row * rows + 1, dtype=x.dtype, device="cuda")[1:]
        out.view(rows, row).copy_(x)
        return out

    def moments(n):
        return [Moment8.zeros(n, "cuda") if bits == 8 else torch.zeros(n, device="cuda") for _ in range(2)]
    (p, grad), ms, ml = [spread(x) for x in small], moments(row), moments(row * rows)
    ws, wl = ([small[0].float().clone()], [spread(small[0].float())]) if master else (None, None)
    for step in (1, 2):
        adamw_step([small[0]], [small[1]], [ms[0]], [ms[1]], step=step, masters=ws, **HYPER)
        adamw_step([p], [grad], [ml[0]], [ml[1]], step=step, masters=wl, **HYPER)
    pairs = [(p, small[0])] + ([(wl[0], ws[0])] if master else [])
    if bits == 8:
        lv, sv = moment8_values([ml[0]], [ml[1]]), moment8_values([ms[0]], [ms[1]])
        pairs += [(a[0], b[0]) for a, b in zip(lv, sv)] + [(a, b) for k in range(2) for a, b in zip(ml[k], ms[k])]
    else:
        pairs += list(zip(ml, ms))
    for long, one in pairs:
        assert (long.view(rows, -1) == one).all()
    torch.cuda.empty_cache()
