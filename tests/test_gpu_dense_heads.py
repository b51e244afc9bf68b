"""The heads on the package's own dense side (CafeCTRHead / CafeCTRModel with dense_ops="hip"): the same losses as torch's
heads, the layers' calls in their order, training with AdamW eagerly, from a checkpoint and captured in a graph."""
import copy
import gc
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(__file__))
from cpu_pipeline import CpuPipeline  # noqa: E402

pytestmark = pytest.mark.gpu
COUNTS = [4000, 197, 25000, 800, 12000, 161]
KINDS = [("dlrm", 13), ("dlrm", 0), ("wdl", 13), ("wdl", 0), ("dcn", 13), ("dcn", 0)]


def head(kind, dense, **kw):
    from cafe_amd.ctr_models import CafeCTRHead
    torch.manual_seed(3)
    return CafeCTRHead(kind, 6, 16, dense, ln_bot=[dense, 32, 16] if dense else None, ln_top=[0, 64, 32, 1], seed=5, **kw)


def inputs(dense, b=200, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.rand(b, dense, device="cuda", generator=g) if dense else None,
            torch.randn(6, b, 16, device="cuda", generator=g) * 0.3, torch.randn(b, 1, device="cuda", generator=g) / b)


@pytest.mark.parametrize("kind,dense_dim", KINDS)
def test_losses_match_the_torch_head(kind, dense_dim, oracle_mod):
    """As the parity test of the torch heads holds them to a CPU twin: per-step losses within 1e-5 relative (float32 sums in
    two orders differ by a few 1e-7 per layer), sketch decisions equal."""
    from cafe_amd.ctr_models import CafeCTRModel
    D, B, lr, thr, F = 16, 256, 0.5, 3, len(COUNTS)
    torch.manual_seed(7)
    model = CafeCTRModel(kind, COUNTS, D, dense_dim=dense_dim, compress_rate=0.05, hash_rate=0.3, threshold=thr,
                         ln_bot=[dense_dim, 32, D] if dense_dim else None, ln_top=[0, 64, 32, 1], seed=5, dense_ops="hip")
    dev = model.embedding.device
    twin = copy.deepcopy(model.head).cpu()
    twin.dense_ops = "torch"
    cpu = CpuPipeline(oracle_mod, model.embedding, thr, 1, 1.0000005)
    opt, opt_c = torch.optim.SGD(model.head.parameters(), lr=lr), torch.optim.SGD(twin.parameters(), lr=lr)
    rng = np.random.default_rng(3)
    for step in range(6):
        ids = np.stack([(rng.zipf(1.1, B) - 1) % n for n in COUNTS]).astype(np.int64)
        ids[0] = np.maximum(ids[0], 1)
        dense = torch.from_numpy(rng.random((B, dense_dim)).astype(np.float32)) if dense_dim else None
        y = torch.from_numpy((rng.random((B, 1)) < 0.25).astype(np.float32))
        loss = model.train_step(None if dense is None else dense.to(dev), torch.from_numpy(ids).to(dev), y.to(dev), opt, lr)
        emb = torch.from_numpy(cpu.forward(ids)).requires_grad_(True)
        opt_c.zero_grad(set_to_none=True)
        loss_c = torch.nn.functional.binary_cross_entropy(twin(dense, emb), y)
        loss_c.backward()
        g = emb.grad.numpy()
        ins = cpu.backward_update(ids, g, np.stack([oracle_mod.ref_scores(g[f]) for f in range(F)]), lr, True)
        opt_c.step()
        assert abs(loss.item() - loss_c.item()) <= 1e-5 * abs(loss_c.item()), f"step {step}"
        assert np.array_equal(model.embedding._buf["ins"].cpu().numpy().reshape(F, B), ins), f"step {step}"


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
def test_dlrm_head_against_float64(t):
    """Running error bound through the layers: a product is off by |W| e_in + (2 n + 16) 2^-24 |W| |h|, every stored value
    by half a step of its type; relu and sigmoid do not amplify; a pair's product by e_i |t_j| + e_j |t_i|."""
    h = head("dlrm", 13, dense_ops="hip", dense_dtype=t).cuda()
    dense, emb, _ = inputs(13)
    u, u32 = torch.finfo(t).eps / 2 * 1.01, 2.0 ** -24
    with torch.no_grad():
        got = h(dense, emb).double()

        def layers(seq, v, e):
            for lin, act in zip(list(seq)[::2], list(seq)[1::2]):
                w, b = lin.weight.double(), lin.bias.double()
                z = v @ w.t() + b
                e = e @ w.abs().t() + (2 * w.shape[1] + 16) * u32 * (v.abs() @ w.abs().t() + b.abs())
                v = z.clamp(min=0) if isinstance(act, torch.nn.ReLU) else torch.sigmoid(z)
                e = e + u * (v + e) + 2 ** -20 * (not isinstance(act, torch.nn.ReLU)) + torch.finfo(t).smallest_normal
            return v, e
        x0 = dense.to(t).double()
        x, e = layers(h.bot_l, x0, torch.zeros_like(x0))
        rows = torch.cat([x[:, None], emb.double().transpose(0, 1)], 1)
        er = torch.cat([e[:, None], torch.zeros_like(rows[:, 1:])], 1)
        i, j = torch.tril_indices(7, 7, -1, device="cuda")
        z = (rows[:, i] * rows[:, j]).sum(2)
        ez = (er[:, i] * rows[:, j].abs() + er[:, j] * rows[:, i].abs() + (2 * 16 + 16) * u32 * (rows[:, i] * rows[:, j]).abs()).sum(2)
        want, err = layers(h.top_l, torch.cat([x, z], 1), torch.cat([e, ez + u * (z.abs() + ez)], 1))
    assert ((got - want).abs() <= err).all()


@pytest.mark.parametrize("kind,dense_dim", KINDS)
def test_gradients_reach_every_parameter_and_row(kind, dense_dim):
    """Every parameter and embedding row gets the gradient that float64 autograd gives the same head.  float32 only: in 16
    bits a relu's input near 0 may take the other side, which no rounding bound covers (the next test compares bits).
    Tolerance (two-norm): at most eight products in a row in either direction, of at most 112 terms, (2 112 + 16) 2^-24 each:
    1.2e-4."""
    h = head(kind, dense_dim, dense_ops="hip").cuda()
    twin = copy.deepcopy(h).double()
    twin.dense_ops = "torch"
    dense, emb, dout = inputs(dense_dim)
    e1, e2 = emb.clone().requires_grad_(), emb.double().requires_grad_()
    h(dense, e1).backward(dout)
    twin(dense.double() if dense_dim else None, e2).backward(dout.double())
    for (n, a), b in zip([("emb", e1)] + list(h.named_parameters()), [e2] + list(twin.parameters())):
        off = float((a.grad.double() - b.grad).norm() / b.grad.norm().clamp(min=1e-30))
        assert off <= 1.2e-4, (n, off)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
def test_dlrm_step_is_its_calls_in_order(t):
    """The head's forward and backward, bit for bit, written out with linear_forward, dot_interaction and linear_backward."""
    from cafe_amd.interact import dot_interaction
    from cafe_amd.linear import linear_backward, linear_forward
    h = head("dlrm", 13, dense_ops="hip", dense_dtype=t).cuda()
    dense, emb, dout = inputs(13)
    e = emb.clone().requires_grad_()
    out = h(dense, e)
    out.backward(dout)

    def forward(seq, v):
        kept = []
        for lin, act in zip(list(seq)[::2], list(seq)[1::2]):
            name = "relu" if isinstance(act, torch.nn.ReLU) else "sigmoid"
            y, k = linear_forward(v, lin.weight, lin.bias, name)
            kept.append((v, lin, k, name))
            v = y
        return v, kept

    def backward(kept, g):
        for v, lin, k, name in reversed(kept):
            g, dw, db = linear_backward(g, v, lin.weight, k, name)
            assert torch.equal(lin.weight.grad, dw) and torch.equal(lin.bias.grad, db)
        return g
    x, bottom = forward(h.bot_l, dense.to(t))
    xl, el = x.detach().requires_grad_(), emb.clone().requires_grad_()
    z = dot_interaction(xl, el, dtype=t)
    y, top = forward(h.top_l, z.detach())
    assert torch.equal(y.float(), out.detach())
    dx, de = torch.autograd.grad(z, [xl, el], backward(top, dout.to(t)))
    backward(bottom, dx)
    same = torch.equal(de, e.grad)
    assert same


@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoint_with_the_optimizer(tmp_path, bits):
    """Model, plain tables, sketch and AdamW state through the driver's checkpoint: everything equal, and the next step's
    loss too."""
    from cafe_amd import train
    from cafe_amd.ctr_models import CafeCTRModel

    def make():
        torch.manual_seed(1)
        m = CafeCTRModel("dlrm", COUNTS + [40], 16, compress_rate=0.05, threshold=3, ln_bot=[13, 32, 16], ln_top=[0, 64, 1], seed=5,
                         dense_ops="hip", dense_dtype=torch.bfloat16)
        return m, train.make_optimizer("adamw8bit" if bits == 8 else "adamw", m.dense_parameters(), 1e-3)
    rng = np.random.default_rng(0)
    batches = []
    for _ in range(5):
        ids = np.stack([np.maximum((rng.zipf(1.1, 128) - 1) % n, 1) for n in COUNTS + [40]]).astype(np.int64)
        batches.append((torch.rand(128, 13).cuda(), torch.from_numpy(ids).cuda(), (torch.rand(128, 1) < 0.3).float().cuda()))
    m, opt = make()
    for b in batches[:4]:
        m.train_step(*b, opt, 0.1)
    path = str(tmp_path / "ck.pt")
    train.save_checkpoint(path, m, 4, opt)
    m2, opt2 = make()
    assert train.load_checkpoint(path, m2, opt2) == 4
    for p, q in zip(m.dense_parameters(), m2.dense_parameters()):
        assert torch.equal(p, q)
        a, b = opt.state[p], opt2.state[q]
        assert a.keys() == b.keys() and ("master" in a) == (p.dtype == torch.bfloat16)
        assert all(torch.equal(a[k], b[k]) and a[k].dtype == b[k].dtype if isinstance(a[k], torch.Tensor) else a[k] == b[k] for k in a)
    assert torch.equal(m.train_step(*batches[4], opt, 0.1), m2.train_step(*batches[4], opt2, 0.1))


def test_driver_options(capsys):
    """The driver with the package's dense side in bfloat16 and 8-bit AdamW."""
    from cafe_amd import train
    m = train.main(["--model", "wdl", "--workload", "cfg5", "--mini-batch-size", "256", "--num-batches", "4", "--print-freq", "2",
                    "--dense-ops", "hip", "--dense-dtype", "bf16", "--optimizer", "adamw8bit", "--dense-learning-rate", "0.001"])
    assert m.head.dense_ops == "hip" and next(m.head.parameters()).dtype == torch.bfloat16
    losses = [float(line.split("loss ")[1].split()[0]) for line in capsys.readouterr().out.splitlines() if "loss " in line]
    assert len(losses) == 2 and all(np.isfinite(losses))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind", ["dlrm", "wdl"])
def test_a_captured_training_step(kind, bits):
    """Forward, backward and AdamW of a head in one graph: every replay equals the eager step of a second copy."""
    from cafe_amd.adamw import AdamW
    dense, emb, dout = inputs(13)
    dense, emb = dense.clone(), emb.requires_grad_()

    def build():
        h = head(kind, 13, dense_ops="hip", dense_dtype=torch.bfloat16).cuda()
        return h, AdamW(h.parameters(), lr=1e-2, state_bits=bits, capturable=True)

    def step(h, opt, e):
        opt.zero_grad(set_to_none=True)
        out = h(dense, e)
        grads = torch.autograd.grad(out, [e] + list(h.parameters()), dout)
        for p, g in zip(h.parameters(), grads[1:]):
            p.grad = g
        opt.step()
        return out.detach(), grads[0]
    h1, o1 = build()
    h2, o2 = build()
    e2 = emb.detach().clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(h1, o1, emb)
    torch.cuda.current_stream().wait_stream(side)
    step(h2, o2, e2)
    gc.collect()                                                # a collected model frees device memory, which a capture forbids
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(h1, o1, emb)
    for k in range(4):
        nd, ne, ng = inputs(13, seed=10 + k)
        dense.copy_(nd); dout.copy_(ng)
        with torch.no_grad():
            emb.copy_(ne); e2.copy_(ne)
        graph.replay()
        want = step(h2, o2, e2)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), k
        assert all(torch.equal(p, q) for p, q in zip(h1.parameters(), h2.parameters())), k
