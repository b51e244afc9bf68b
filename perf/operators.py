"""The dense-side operators of the package at the sizes its models use them, each beside its plain form.

    linear / linear_backward   y = act(x W^T + b) + residual and its gradients      cafe_amd.linear
    dot_interaction            pairwise products of a sample's feature rows          cafe_amd.interact
    adamw_step                 one AdamW step over many tensors, 32- or 8-bit states cafe_amd.adamw

`own` False: run() computes the plain form with elementary torch operations in float32 and rounds once at the end.
`own` True: run() makes the calls a user makes.  exact() restates the definitions in float64."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 256                      # elements of a moment that share one exponent


# ------------------------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------------------------
def _linear(name, do, m, k, n, act, dtype, bias=True, residual=False, pad=0):
    return {"name": name, "op": "linear", "do": do, "m": m, "k": k, "n": n, "act": act, "dtype": dtype, "bias": bias,
            "residual": residual, "pad": pad}


def _interact(name, do, batch, fields, dim, dense, itself, emb, dtype):
    return {"name": name, "op": "interact", "do": do, "batch": batch, "fields": fields, "dim": dim, "dense": dense,
            "itself": itself, "emb": emb, "dtype": dtype}


def _adamw(name, sizes, dtype, bits, master):
    return {"name": name, "op": "adamw", "sizes": sizes, "dtype": dtype, "bits": bits, "master": master}


def _mlp(widths):
    """The tensors of an MLP as x-separated shapes: weight [out, in] and bias [out] of every layer."""
    return ["%dx%d %d" % (o, i, o) for i, o in zip(widths, widths[1:])]


def listed():
    dlrm128 = " ".join(_mlp([13, 512, 256, 128]) + _mlp([479, 1024, 1024, 512, 256, 1]))
    dlrm16 = " ".join(_mlp([13, 512, 256, 64, 16]) + _mlp([367, 512, 256, 1]))
    wdl128 = " ".join(_mlp([3341, 1]) + _mlp([3341, 256, 256, 1]))
    return [
        # one request scored by a DLRM: its first top layer
        _linear("linear_one_row_bf16", "forward", 1, 479, 1024, "relu", "bf16"),
        # the same layer under the training batch, at the framework's default type
        _linear("linear_top_f32", "forward", 8192, 479, 1024, "relu", "f32"),
        # WDL's last layer: the deep part's sigmoid with the wide part's logit added
        _linear("linear_deep_plus_wide_f32", "forward", 8192, 256, 1, "sigmoid", "f32", residual=True),
        # gradients of DLRM's widest layer, from the output its forward kept
        _linear("linear_gradients_f32", "backward", 8192, 1024, 1024, "relu", "f32"),
        # the smallest training batch: a residual block of a narrow head
        _linear("linear_step_small_f16", "step", 128, 367, 367, "gelu", "f16", residual=True),
        # WDL's first layer at D = 128, the largest batch: forward and backward
        _linear("linear_step_wide_bf16", "step", 16384, 3341, 256, "silu", "bf16"),
        # one request without dense features (22 fields, D = 16)
        _interact("interact_one_row_f32", "forward", 1, 22, 16, False, False, "f32", "f32"),
        # training step at D = 128: forward and backward
        _interact("interact_step_f32", "step", 8192, 26, 128, True, False, "f32", "f32"),
        # bf16 head on float32 embedding rows (D = 16), the largest batch
        _interact("interact_step_bf16", "step", 16384, 26, 16, True, True, "f32", "bf16"),
        # the optimizer step of a small DLRM head: launch latency
        _adamw("adamw_small_head_f32", dlrm16, "f32", 32, False),
        # the DLRM head at D = 128 with 8-bit states
        _adamw("adamw_head_8bit_f32", dlrm128, "f32", 8, False),
        # WDL head in bf16 with float32 master weights, and plain tables of tens of millions of values, 8-bit states
        _adamw("adamw_tables_8bit_bf16", wdl128 + " 130001x128 1000003x16 77777x33 7", "bf16", 8, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = max((work(c) for c in listed()), key=lambda w: w["flops"])
    while True:
        op = rng.choice(["linear", "linear", "interact", "adamw"])
        if op == "linear":
            do = rng.choice(["forward", "backward", "step"])
            act = rng.choice(["none", "relu", "sigmoid", "gelu", "silu"])
            if do == "step" and act == "relu":
                do = "backward"         # from a kept output: the sign of a sum at 0 differs from one order of summation to another
            c = _linear("", do, _log(rng, 1, 16384), _log(rng, 1, 4096), _log(rng, 1, 2048), act,
                        rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.8, rng.random() < 0.3 and do != "backward",
                        rng.choice([0, 0, 1, 3, 16]))
        elif op == "interact":
            c = _interact("", rng.choice(["forward", "step"]), _log(rng, 1, 16384), rng.randint(1, 40), _log(rng, 1, 200),
                          rng.random() < 0.7, rng.random() < 0.4, "f32", rng.choice(["f32", "bf16", "f16"]))
            if c["fields"] == 1 and not c["dense"] and not c["itself"]:
                continue                # no pair: nothing comes back
            if rng.random() < 0.3:
                c["emb"] = c["dtype"]
            if c["batch"] * (c["fields"] + 1) * c["dim"] > 8192 * 27 * 128:
                continue
        else:
            sizes = ["x".join(str(v) for v in ([_log(rng, 1, 4096), _log(rng, 1, 1024)] if rng.random() < 0.6 else
                                               [_log(rng, 1, 65536)])) for _ in range(rng.randint(1, 16))]
            c = _adamw("", " ".join(sizes), rng.choice(["f32", "bf16", "f16"]), rng.choice([8, 32]), False)
            c["master"] = c["dtype"] != "f32" and rng.random() < 0.6
        w = work(c)
        if w["flops"] <= most["flops"] and w["bytes"] <= 4e8:
            del c["name"]
            return c


# ------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------
def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["sizes"].split()]


def _encode(v, second):
    """A float32 tensor as 8-bit codes and one exponent byte per block of 256 consecutive values.

    The block's exponent E is that of its largest finite magnitude (at least -126), values are scaled by 2^-E into
    [0, 2) and rounded, to nearest with ties to even, to a small floating format whose top binade is [1, 2): the
    first moment (signed) has 4 exponent and 3 mantissa bits, the second (never negative) 5 and 3.  A second moment
    above 0 never becomes 0.  Code 0x80 of the first moment stands for a value that is not finite (read as NaN),
    code 0xff of the second (read as infinity); the exponent is stored plus 127."""
    flat = v.reshape(-1)
    n = flat.numel()
    x = torch.nn.functional.pad(flat, (0, -n % BLOCK)).view(-1, BLOCK)
    mag = x.abs()
    ok = torch.isfinite(x)
    top = torch.where(ok, mag, torch.zeros_like(mag)).amax(1, keepdim=True)
    e = (torch.frexp(top)[1] - 1).clamp(min=-126)
    e = torch.where(top > 0, e, torch.full_like(e, -126))
    a = torch.where(ok, mag, torch.zeros_like(mag)).double() * torch.exp2(-e.double())
    low = -30 if second else -14                        # exponent of the smallest normal code
    b = torch.where(a > 0, torch.frexp(a)[1] - 1, torch.full_like(e, low)).clamp(min=low)
    steps = torch.round(a * torch.exp2((3 - b).double())).long()          # in units of 2^(b - 3)
    code = steps + 8 * (b.long() - low)                 # steps 8..16 of binade b; below 8 only at b == low
    code = code.clamp(max=0xfe if second else 0x7f)
    if second:
        code = torch.where((code == 0) & (mag > 0), torch.ones_like(code), code)
        code = torch.where(ok, code, torch.full_like(code, 0xff))
    else:
        code = torch.where((x < 0) & (code > 0), code + 0x80, code)
        code = torch.where(ok, code, torch.full_like(code, 0x80))
    return code.to(torch.uint8).view(-1)[:n].contiguous(), (e + 127).to(torch.uint8).view(-1)


def _decode(codes, exponents, second):
    """The float32 values that _encode's bytes stand for."""
    c = codes.long()
    low = -30 if second else -14
    mag = c if second else c & 0x7f
    field = mag >> 3
    steps = torch.where(field > 0, 8 + (mag & 7), mag & 7)
    scale = torch.where(field > 0, field - 1, field) + (low - 3)
    e = exponents.long().sub(127).repeat_interleave(BLOCK)[:c.numel()]
    v = (steps.double() * torch.exp2((scale + e).double())).float()
    if second:
        return torch.where(c == 0xff, torch.full_like(v, math.inf), v)
    v = torch.where(c > 0x80, -v, v)
    return torch.where(c == 0x80, torch.full_like(v, math.nan), v)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "linear":
        return _prepare_linear(case, g)
    if case["op"] == "interact":
        return _prepare_interact(case, g)
    return _prepare_adamw(case, g)


def _randn(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def _prepare_linear(case, g):
    m, k, n, t = case["m"], case["k"], case["n"], DTYPES[case["dtype"]]
    step = case["do"] == "step"
    s = dict(case)
    s["x"] = _randn(g, m, k + case["pad"]).to(t)[:, :k].requires_grad_(step)
    s["w"] = (_randn(g, n, k) * math.sqrt(2.0 / (n + k))).to(t).requires_grad_(step)        # create_mlp's scale
    s["b"] = (_randn(g, n) * math.sqrt(1.0 / n)).to(t).requires_grad_(step) if case["bias"] else None
    s["r"] = _randn(g, m, n).to(t).requires_grad_(step) if case["residual"] else None
    if case["do"] != "forward":
        s["dy"] = _randn(g, m, n).to(t)
    if case["do"] == "backward":        # what the forward keeps: relu's output, the value before the activation otherwise
        z = _randn(g, m, n)
        s["saved"] = None if case["act"] == "none" else (z.clamp(min=0) if case["act"] == "relu" else z).to(t)
    return s


def _pairs(nf, itself):
    return nf * (nf + 1) // 2 if itself else nf * (nf - 1) // 2


def _prepare_interact(case, g):
    b, f, d = case["batch"], case["fields"], case["dim"]
    step = case["do"] == "step"
    s = dict(case)
    s["x"] = _randn(g, b, d).to(DTYPES[case["dtype"]]).requires_grad_(step) if case["dense"] else None
    s["emb"] = (_randn(g, f, b, d) * 0.3).to(DTYPES[case["emb"]]).requires_grad_(step)
    if step:
        width = _pairs(f + int(case["dense"]), case["itself"]) + (d if case["dense"] else 0)
        s["dout"] = _randn(g, b, width).to(DTYPES[case["dtype"]])
    return s


def _prepare_adamw(case, g):
    """Weights, gradients and moments of a run in progress: gradient sizes differ from tensor to tensor, and inside one
    (rows of ids that are hardly seen), the second moments with them."""
    t = DTYPES[case["dtype"]]
    s = dict(case, step=100, p=[], g=[], m=[], v=[], w=[])
    for shape in _shapes(case):
        scale = torch.exp(_randn(g, 1) - 5.0)
        rows = torch.exp(_randn(g, shape[0], *([1] * (len(shape) - 1))))
        w = _randn(g, *shape) * 0.05
        grad = _randn(g, *shape) * scale * rows
        m = _randn(g, *shape) * scale * rows * 0.3
        v = (scale * rows).square() * torch.exp(0.5 * _randn(g, *shape))
        s["p"].append(w.to(t))
        s["g"].append(grad.to(t))
        s["m"].append(_encode(m, False) if case["bits"] == 8 else m)
        s["v"].append(_encode(v, True) if case["bits"] == 8 else v)
        s["w"].append(w if case["master"] else None)
    return s


# ------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return {"linear": _own_linear, "interact": _own_interact, "adamw": _own_adamw}[state["op"]](state)
    with torch.no_grad():
        return {"linear": _plain_linear, "interact": _plain_interact, "adamw": _plain_adamw}[state["op"]](state)


def _own_linear(s):
    from cafe_amd.linear import linear, linear_backward
    if s["do"] == "forward":
        return linear(s["x"], s["w"], s["b"], s["act"], s["r"])
    if s["do"] == "backward":
        dx, dw, db = linear_backward(s["dy"], s["x"], s["w"], s["saved"], s["act"])
        return {"dx": dx, "dw": dw, "db": db}
    y = linear(s["x"], s["w"], s["b"], s["act"], s["r"])
    keys = [k for k in ("x", "w", "b", "r") if s[k] is not None]
    grads = torch.autograd.grad(y, [s[k] for k in keys], s["dy"])
    return dict(zip(["y"] + ["d" + k for k in keys], (y,) + grads))


def _own_interact(s):
    from cafe_amd.interact import dot_interaction
    y = dot_interaction(s["x"], s["emb"], itself=s["itself"], dtype=DTYPES[s["dtype"]])
    if s["do"] == "forward":
        return y
    keys = [k for k in ("x", "emb") if s[k] is not None]
    grads = torch.autograd.grad(y, [s[k] for k in keys], s["dout"])
    return dict(zip(["y"] + ["d" + k for k in keys], (y,) + grads))


HYPER = {"lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01}


def _own_adamw(s):
    from cafe_amd.adamw import Moment8, adamw_step, moment8_values
    s["step"] += 1
    masters = s["w"] if s["master"] else None
    if s["bits"] == 32:
        adamw_step(s["p"], s["g"], s["m"], s["v"], step=s["step"], masters=masters, **HYPER)
        m, v = s["m"], s["v"]
    else:
        m8, v8 = [Moment8(*t) for t in s["m"]], [Moment8(*t) for t in s["v"]]
        adamw_step(s["p"], s["g"], m8, v8, step=s["step"], masters=masters, **HYPER)
        m, v = moment8_values(m8, v8)
    return {"p": s["p"], "m": [t.reshape(-1) for t in m], "v": [t.reshape(-1) for t in v], "w": masters or []}


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    e = torch.exp(-z.abs())
    sig = torch.where(z > 0, 1 / (1 + e), e / (1 + e))
    if act == "sigmoid":
        return e / ((1 + e) * (1 + e))
    if act == "silu":
        return sig * (1 + z * (1 - sig))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi)
    return torch.ones_like(z)


def _plain_linear(s):
    t = DTYPES[s["dtype"]]
    x, w = s["x"].float(), s["w"].float()
    if s["do"] != "backward":
        z = torch.matmul(x, w.t())
        z = z + s["b"].float() if s["b"] is not None else z
        y = _act(z, s["act"])
        y = y + s["r"].float() if s["r"] is not None else y
        if s["do"] == "forward":
            return y.to(t)
    else:
        z = s["saved"].float() if s["saved"] is not None else None
    dy = s["dy"].float()
    dz = dy * _act_slope(z, s["act"]) if s["act"] != "none" else dy
    grads = {"dx": torch.matmul(dz, w).to(t), "dw": torch.matmul(dz.t(), x).to(t), "db": dz.sum(0).to(t)}
    if s["do"] == "backward":
        return grads
    out = {"y": y.to(t), **grads}
    if s["b"] is None:
        del out["db"]
    if s["r"] is not None:
        out["dr"] = s["dy"]
    return out


def _plain_interact(s):
    f, t = s["emb"].shape[0], DTYPES[s["dtype"]]
    rows = s["emb"].float().transpose(0, 1)
    x = s["x"].float() if s["x"] is not None else None
    rows = rows if x is None else torch.cat([x[:, None, :], rows], 1)
    nf, d = rows.shape[1], rows.shape[2]
    rows = rows.contiguous()
    z = torch.bmm(rows, rows.transpose(1, 2).contiguous())
    i, j = torch.tril_indices(nf, nf, 0 if s["itself"] else -1, device=rows.device)
    flat = z[:, i, j]
    y = (flat if x is None else torch.cat([x, flat], 1)).to(t)
    if s["do"] == "forward":
        return y
    dout = s["dout"].float()
    dz = torch.zeros_like(z)
    dz[:, i, j] = dout[:, (d if x is not None else 0):]
    drows = torch.bmm(dz + dz.transpose(1, 2), rows)
    out = {"y": y}
    if x is not None:
        out["dx"] = (drows[:, 0] + dout[:, :d]).to(t)
        drows = drows[:, 1:]
    out["demb"] = drows.transpose(0, 1).contiguous().to(s["emb"].dtype)
    assert out["demb"].shape[0] == f
    return out


def _plain_adamw_one(s, k):
    """Tensor k's step: the order of operations of the definition, each rounded to float32."""
    b1, b2 = HYPER["betas"]
    g = s["g"][k].float()
    m = _decode(*s["m"][k], False).view(g.shape) if s["bits"] == 8 else s["m"][k]
    v = _decode(*s["v"][k], True).view(g.shape) if s["bits"] == 8 else s["v"][k]
    p = s["w"][k] if s["master"] else s["p"][k].float()
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    denom = torch.sqrt(v) / math.sqrt(1 - b2 ** s["step"]) + HYPER["eps"]
    p = p * (1 - HYPER["lr"] * HYPER["weight_decay"]) - (m / denom) * (HYPER["lr"] / (1 - b1 ** s["step"]))
    if s["bits"] == 8:
        m8, v8 = _encode(m, False), _encode(v, True)
        [dst.copy_(src) for dst, src in zip(s["m"][k] + s["v"][k], m8 + v8)]
        m, v = _decode(*m8, False), _decode(*v8, True)
    else:
        s["m"][k].copy_(m)
        s["v"][k].copy_(v)
    if s["master"]:
        s["w"][k].copy_(p)
    s["p"][k].copy_(p)
    return m.reshape(-1), v.reshape(-1)


def _plain_adamw(s):
    s["step"] += 1
    mv = [_plain_adamw_one(s, k) for k in range(len(s["p"]))]
    return {"p": s["p"], "m": [a for a, _ in mv], "v": [b for _, b in mv], "w": s["w"] if s["master"] else []}


# ------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "linear":
        m, k, n, e = case["m"], case["k"], case["n"], SIZE[case["dtype"]]
        fwd = m * k + n * k + n * case["bias"] + m * n * (1 + case["residual"])
        kept = m * n if case["act"] != "none" else 0
        grads = m * k + n * k + n * (1 if case["do"] == "backward" else case["bias"])
        if case["do"] == "forward":
            return {"bytes": e * fwd, "flops": 2 * m * n * k}
        if case["do"] == "backward":
            return {"bytes": e * (m * k + n * k + m * n + kept + grads), "flops": 4 * m * n * k}
        return {"bytes": e * (fwd + m * n + grads), "flops": 6 * m * n * k}
    if case["op"] == "interact":
        b, f, d, dense = case["batch"], case["fields"], case["dim"], int(case["dense"])
        pairs = _pairs(f + dense, case["itself"])
        rows = b * d * (f * SIZE[case["emb"]] + dense * SIZE[case["dtype"]])
        out = b * (pairs + dense * d) * SIZE[case["dtype"]]
        if case["do"] == "forward":
            return {"bytes": rows + out, "flops": 2 * b * pairs * d}
        return {"bytes": 2 * (rows + out), "flops": 6 * b * pairs * d}
    n = sum(math.prod(s) for s in _shapes(case))
    e = SIZE[case["dtype"]]
    states = 16 if case["bits"] == 32 else 4 + 8 + 8 / BLOCK            # 8 bits: the values they stand for are written too
    return {"bytes": int(n * (3 * e + (8 if case["master"] else 0) + states)), "flops": 12 * n}


# ------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"linear": _exact_linear, "interact": _exact_interact, "adamw": _exact_adamw}[case["op"]](s)


def _exact_linear(s):
    x, w = s["x"].double(), s["w"].double()
    one = torch.ones((), dtype=torch.float64, device=x.device)
    phi = lambda z: 0.5 * torch.special.erfc(-z / math.sqrt(2.0))                            # noqa: E731
    value = {"none": lambda z: z, "relu": lambda z: torch.maximum(z, 0 * one), "sigmoid": torch.special.expit,
             "silu": lambda z: z * torch.special.expit(z), "gelu": lambda z: z * phi(z)}[s["act"]]
    slope = {"none": lambda z: one, "relu": lambda z: torch.heaviside(z, 0 * one),
             "sigmoid": lambda z: torch.special.expit(z) * torch.special.expit(-z),
             "silu": lambda z: torch.special.expit(z) + z * torch.special.expit(z) * torch.special.expit(-z),
             "gelu": lambda z: phi(z) + z * torch.exp(-z ** 2 / 2) / math.sqrt(2 * math.pi)}[s["act"]]
    out = {}
    z = s["saved"].double() if s.get("saved") is not None else None
    if s["do"] != "backward":
        z = torch.nn.functional.linear(x, w, None if s["b"] is None else s["b"].double())
        y = value(z) + (0 * one if s["r"] is None else s["r"].double())
        if s["do"] == "forward":
            return y
        out["y"] = y
        if s["r"] is not None:
            out["dr"] = s["dy"].double()
    dz = s["dy"].double() * (one if z is None else slope(z))
    out["dx"] = dz @ w
    out["dw"] = (x.t() @ dz).t()
    if s["do"] == "backward" or s["b"] is not None:
        out["db"] = torch.ones(1, dz.shape[0], dtype=dz.dtype, device=dz.device).mm(dz)[0]
    return out


def _exact_interact(s):
    """Pair by pair of fields: z_ij = <t_i, t_j>, and from dz_ij to the two rows' gradients."""
    t = [e.double() for e in s["emb"]]
    if s["x"] is not None:
        t = [s["x"].double()] + t
    pairs = [(i, j) for i in range(len(t)) for j in range(i + int(s["itself"]))]
    lead = [] if s["x"] is None else [t[0]]
    z = [(t[i] * t[j]).sum(1, keepdim=True) for i, j in pairs]
    y = torch.cat(lead + z, 1)
    if s["do"] == "forward":
        return y
    dout = s["dout"].double()
    at = lead[0].shape[1] if lead else 0
    grads = [torch.zeros_like(v) for v in t]
    if lead:
        grads[0] += dout[:, :at]
    for q, (i, j) in enumerate(pairs):
        dz = dout[:, at + q:at + q + 1]
        grads[i] += dz * t[j]
        grads[j] += dz * t[i]
    if lead:
        return {"y": y, "dx": grads[0], "demb": torch.stack(grads[1:])}
    return {"y": y, "demb": torch.stack(grads)}


def _exact_adamw(s):
    """8-bit moments have no value here: one next to a rounding border goes either way with the last bit of a sum."""
    lr, (b1, b2), step = HYPER["lr"], HYPER["betas"], s["step"] + 1
    out = {"p": [], "m": [], "v": [], "w": []}
    for k, g in enumerate(s["g"]):
        g = g.double()
        eight = s["bits"] == 8
        m = (_decode(*s["m"][k], False) if eight else s["m"][k]).double().view(g.shape)
        v = (_decode(*s["v"][k], True) if eight else s["v"][k]).double().view(g.shape)
        m = torch.lerp(m, g, 1 - b1)
        v = torch.lerp(v, g ** 2, 1 - b2)
        p = (s["w"][k] if s["master"] else s["p"][k]).double()
        p = p - lr * HYPER["weight_decay"] * p - lr * (m / (1 - b1 ** step)) / ((v / (1 - b2 ** step)) ** 0.5 + HYPER["eps"])
        out["p"].append(p)
        out["m"].append(None if eight else m.reshape(-1))
        out["v"].append(None if eight else v.reshape(-1))
        if s["master"]:
            out["w"].append(p)
    return out
