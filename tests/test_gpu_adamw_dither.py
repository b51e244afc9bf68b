"""8-bit moments over a run of steps: right on average, where rounding to nearest leaves them standing still; the codes, bit
for bit, from the definition of the rounding.

Tolerances of the long runs.  A rounding that is unbiased leaves the mean of v in place: v is a linear recursion.  One code
step s is at most v / 8, and a step of AdamW moves v by some (1 - b2) v, so a rounding adds a variance of at most
(1 - b2) v s <= (1 - b2) v^2 / 8, and forgets at 2 (1 - b2): together v^2 / 16, a quarter of v at most (while v falls tenfold or
more, what was added before weighs more: half of v).  The mean over 4096 values is then good to 0.5 / 64 = 0.8 %; 5 % is six
times that.  The first eight steps are off by half a code step, 1 / 16, and forgotten.  Updates go with v^-1/2, whose mean is
1 + 3 / 8 of the relative variance: 2 % (9 % while v falls), m's own noise averages out: 10 % of the mean distance."""
import gc

import pytest
import torch

from cafe_amd.adamw import AdamW, Moment8, adamw_step, moment8_values

pytestmark = pytest.mark.gpu
N = 4096
MASK = 0xFFFFFFFF


def scramble(h):
    h = h ^ (h >> 16)
    h = (h * 0x6A09E667) & MASK
    h = h ^ (h >> 15)
    h = (h * 0xBB67AE85) & MASK
    return h ^ (h >> 16)


def bits(step, n, start=0):
    """The hash of values start .. start + n - 1 (start a multiple of 8, no multiple of 2^32 between) in step `step`."""
    key = scramble(scramble(torch.tensor((step * 0x9E3779B9 + (step >> 32)) & MASK)) + (start >> 32) & MASK)
    return scramble(((torch.arange(n) + (start & MASK)) * 0x9E3779B9 + key) & MASK)


def encode(x, second, h):
    """Codes and exponents of float32 values: down or up a code, up where the fraction of the step and 20 bits reach 1."""
    low, limit = (-30, 1.75) if second else (-14, 1.875)
    x = x.detach().cpu().double().reshape(-1)
    up = ((h if second else (h << 16 | h >> 16) & MASK) >> 12).double() * 2.0 ** -20
    codes, exps = [], []
    for k in range(0, x.numel(), 256):
        b = x[k:k + 256]
        top = b.abs().max()
        e = int(torch.frexp(top)[1]) - 1
        e += bool(top * 2.0 ** -e >= limit)
        a = b.abs() * 2.0 ** -e
        binade = torch.where(a > 0, torch.frexp(a)[1] - 1, torch.full((), low, dtype=torch.int32)).clamp(min=low)
        c = (torch.floor(a * torch.exp2(3.0 - binade) + up[k:k + 256]) + 8 * (binade - low)).long()
        c = torch.where((c == 0) & (b > 0), 1, c) if second else torch.where((b < 0) & (c > 0), c + 128, c)
        codes.append(c)
        exps.append(e + 127)
    return torch.cat(codes).to(torch.uint8).cuda(), torch.tensor(exps, dtype=torch.uint8, device="cuda")


def values(n, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(n, device="cuda", generator=g) * torch.exp(2 * torch.randn(n, device="cuda", generator=g))


RUNS = {"constant": lambda t, z: torch.ones_like(z), "random": lambda t, z: z,
        "shrinking": lambda t, z: z * (1.0 if t < 1000 else 0.1), "constant, then shrinking": lambda t, z: torch.full_like(z, 1.0 if t < 1000 else 0.1)}


@pytest.mark.parametrize("kind", list(RUNS))
def test_three_thousand_steps(kind):
    """Against float32 moments; rounded to nearest, v ends at 0.014 to 1.9 of the true one and the distance at 1.6 to 5 times."""
    g = torch.Generator(device="cuda").manual_seed(0)
    scale = torch.exp(0.5 * torch.randn(N, device="cuda", generator=g))
    ps = [torch.nn.Parameter(torch.zeros(N, device="cuda")) for _ in range(2)]
    opts = [AdamW([p], lr=1e-3, weight_decay=0.0, state_bits=b) for p, b in zip(ps, (8, 32))]
    for t in range(1, 3001):
        grad = RUNS[kind](t, torch.randn(N, device="cuda", generator=g) * scale)
        for p, o in zip(ps, opts):
            p.grad = grad
            o.step()
    st = opts[0].state[ps[0]]
    (m,), (v,) = moment8_values([Moment8(st["exp_avg_codes"], st["exp_avg_exponents"])], [Moment8(st["exp_avg_sq_codes"], st["exp_avg_sq_exponents"])])
    true = opts[1].state[ps[1]]
    assert abs(float((v / true["exp_avg_sq"]).mean()) - 1) <= 0.05
    assert abs(float(ps[0].detach().abs().mean() / ps[1].detach().abs().mean()) - 1) <= 0.1


@pytest.mark.parametrize("step", [9, 1000, 2 ** 33 + 5])
@pytest.mark.parametrize("on_device", [False, True])
def test_codes(step, on_device):
    """One step from zero moments, betas chosen so that m = g and v = g^2 in float32: tensors of several sizes in one call."""
    sizes = [1, 7, 256, 257, 5000, 70001]
    gs = [values(n, n) for n in sizes]
    gs[3][:200] = 1.97                                          # a block whose largest is above the largest code
    gs[4][::3] = 0.0
    ms, vs = [[Moment8.zeros(n, "cuda") for n in sizes] for _ in range(2)]
    ps = [torch.zeros(n, device="cuda") for n in sizes]
    d = torch.tensor([step], device="cuda") if on_device else step
    adamw_step(ps, gs, ms, vs, step=1, lr=0.0, betas=(0.0, 0.0), eps=1.0, weight_decay=0.0, dither=d)
    for n, g, m, v in zip(sizes, gs, ms, vs):
        h = bits(step, n)
        for got, want in ((m, encode(g, False, h)), (v, encode(g * g, True, h))):
            assert torch.equal(got.exponents, want[1]) and torch.equal(got.codes, want[0]), n


def test_nothing_is_cut_off_at_the_top():
    """Blocks full of one value between the largest code and the next exponent keep their mean.  A code step is at most an
    eighth of the value, a rounding's standard deviation half of that, the mean's over 2^20 values 6.1e-5: ten times that."""
    n = 1 << 20
    for x in (1.9, 1.99, 1.7, 1.0):
        g = torch.full((n,), x, device="cuda")
        m, v = Moment8.zeros(n, "cuda"), Moment8.zeros(n, "cuda")
        adamw_step([torch.zeros(n, device="cuda")], [g], [m], [v], step=1, lr=0.0, betas=(0.0, 0.0), eps=1.0, weight_decay=0.0, dither=77)
        (gm,), (gv,) = moment8_values([m], [v])
        assert abs(float(gm.double().mean()) - x) <= 6e-4 * x and abs(float(gv.double().mean()) - x * x) <= 6e-4 * x * x


def test_the_first_steps_round_to_nearest_and_groups_do_not_matter():
    sizes = [300, 5000]
    gs = [values(n, n) * 1e-2 for n in sizes]

    def run(dithers, split):
        ps = [torch.zeros(n, device="cuda") for n in sizes]
        ms, vs = [[Moment8.zeros(n, "cuda") for n in sizes] for _ in range(2)]
        for step, d in enumerate(dithers, 1):
            for part in ([[0], [1]] if split else [[0, 1]]):
                pick = lambda ts: [ts[i] for i in part]                                # noqa: E731
                adamw_step(pick(ps), pick(gs), pick(ms), pick(vs), step=step, lr=1e-2, dither=d)
        return ps + [t for m in ms + vs for t in m]
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))                   # noqa: E731
    assert same(run(range(1, 9), False), run([None] * 8, False))
    whole = run(range(1, 30), False)
    assert same(whole, run(range(1, 30), True)) and same(whole, run(range(1, 30), False))
    assert not same(whole, run([None] * 29, False))


def test_indices_past_32_bits():
    """Values behind 2^32 have random bits of their own, those of the definition; so do the pieces of a long tensor."""
    n, far = 2 ** 32 + 1024, 2 ** 32
    row = values(1024, 3).bfloat16()
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    places = (0, 2 ** 31, far)
    for at in places:
        g[at:at + 1024] = row
    p, m, v = torch.zeros_like(g), Moment8.zeros(n, "cuda"), Moment8.zeros(n, "cuda")
    adamw_step([p], [g], [m], [v], step=1, lr=0.0, betas=(0.0, 0.0), eps=1.0, weight_decay=0.0, dither=20)
    f, seen = row.float(), []
    for at in places:
        h = bits(20, 1024, at)
        for got, want in ((m.codes, encode(f, False, h)[0]), (v.codes, encode(f * f, True, h)[0])):
            assert torch.equal(got[at:at + 1024], want), at
        seen.append(m.codes[at:at + 1024].clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[0], seen[2])
    del g, p, m, v
    torch.cuda.empty_cache()


def test_replays_go_on_with_the_device_count():
    """Captured and replayed past the ninth step, among eager work: every replay is the eager step."""
    p = torch.nn.Parameter(values(5000, 1).bfloat16())
    q = torch.nn.Parameter(p.detach().clone())
    opt, ref = AdamW([p], lr=1e-2, state_bits=8, capturable=True), AdamW([q], lr=1e-2, state_bits=8)
    grad = values(5000, 2).bfloat16()
    p.grad, q.grad = grad, grad
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
        with pytest.raises(Exception, match="same random bits"):
            z = torch.zeros(1, device="cuda")
            adamw_step([z], [z], [Moment8.zeros(1, "cuda")], [Moment8.zeros(1, "cuda")], factors=torch.ones(3, device="cuda"), lr=0.1, dither=9)
    for k in range(20):
        grad.copy_(values(5000, 10 + k))
        graph.replay()
        ref.step()
        torch.cuda.synchronize()
        assert torch.equal(p, q), k
        a, b = opt.state[p], ref.state[q]
        assert all(torch.equal(a[x], b[x]) for x in a if isinstance(a[x], torch.Tensor)), k
