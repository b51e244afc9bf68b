"""AdamW over many tensors in one launch (cafe_amd/csrc/cafe_adamw.hip), moments in 32 or 8 bits.

The dense parameters of a head are a dozen tensors between one value and a few million; the reference steps them with
torch.optim.  `AdamW` is a torch.optim.Optimizer; `adamw_step` the step itself over lists of tensors; `moment8_values`
the float32 values that 8-bit moments stand for."""
import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .linear import DTYPE_CODE, launch_on, on_device

BLOCK = 256                     # values that share one exponent


class Moment8(NamedTuple):
    """A moment in 8 bits: a code per value of the flattened tensor and an exponent (plus 127) per 256 of them."""
    codes: torch.Tensor
    exponents: torch.Tensor

    @classmethod
    def zeros(cls, n, device):
        return cls(torch.zeros(n, dtype=torch.uint8, device=device),
                   torch.ones(-(-n // BLOCK), dtype=torch.uint8, device=device))


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _check(tensors, dtype, index, sizes, what):
    """Every tensor of `dtype` on device `index`, contiguous, of the sizes listed (shapes, or numbers of values)."""
    by_shape = sizes and not isinstance(sizes[0], int)
    if not (all([t.dtype is dtype and t.get_device() == index and t.is_contiguous() for t in tensors])
            and [t.shape if by_shape else t.numel() for t in tensors] == sizes):
        for i, (t, n) in enumerate(zip(tensors, sizes)):
            if t.dtype is not dtype or t.get_device() != index or not t.is_contiguous() or (t.shape if by_shape else t.numel()) != n:
                raise ValueError(f"{what}[{i}]: contiguous {dtype} of {n if by_shape else f'{n} values'} on the parameters' device "
                                 f"expected, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _check_moments8(moments, counts, index, what):
    """Moment8 throughout, codes and exponents of the right sizes; returns the lists of both."""
    if not all([type(m) is Moment8 for m in moments]):
        raise ValueError(f"{what}: Moment8 expected beside Moment8")
    codes, exponents = [m[0] for m in moments], [m[1] for m in moments]
    _check(codes, torch.uint8, index, counts, f"{what} codes")
    _check(exponents, torch.uint8, index, [_blocks(n) for n in counts], f"{what} exponents")
    return codes, exponents


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step=None, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
               masters=None, factors=None, dither=None):
    """One AdamW step in place over lists of tensors:

        m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - b1^step) m / (sqrt(v) / sqrt(1 - b2^step) + eps)

    params: contiguous, of one type (float32, bfloat16, float16), on one GPU, no two sharing memory; grads: of the same
    type and shape.  exp_avgs, exp_avg_sqs: float32 tensors of the parameter's shape, or Moment8 throughout.  masters:
    None, or float32 tensors of the parameters' shapes that are updated in their place; the parameters then receive the
    rounded values (a float32 parameter may be its own master).  step: the number of this step, from 1; it is a number of
    the host, so a call under graph capture takes `factors` instead (adamw_tick), a float32 tensor of three on the device.
    dither: for Moment8, the number of this step in a run of them, from 1, or an int64 tensor of one on the device (under
    capture: the tensor that adamw_tick counts in); AdamW always gives it.  From the ninth step on the moments are rounded up
    or down with the probabilities that leave their mean in place, by a hash of this number and a value's index.  Without it
    they are rounded to nearest: right for a single step, but in a run of them v would stand still, since a step changes it by
    less than half a code.  All arithmetic is float32."""
    n = len(params)
    if not (len(grads) == len(exp_avgs) == len(exp_avg_sqs) == n) or (masters is not None and len(masters) != n):
        raise ValueError("params, grads, moments and masters are lists of one length")
    if n == 0:
        return
    first = params[0]
    dtype, index = first.dtype, first.get_device()
    if dtype not in DTYPE_CODE:
        raise ValueError(f"float32, bfloat16 or float16 parameters expected, not {dtype}")
    eight = isinstance(exp_avgs[0], Moment8)
    shapes, counts = [p.shape for p in params], [p.numel() for p in params]
    _check(params, dtype, index, counts, "params")
    if not all([g.layout is torch.strided for g in grads]):
        raise ValueError("grads: dense tensors expected")
    grads = [g if g.is_contiguous() else g.contiguous() for g in grads]             # copies live until the launch is queued
    _check(grads, dtype, index, shapes, "grads")
    zeros = [0] * n
    cols = [[p.data_ptr() for p in params], [g.data_ptr() for g in grads]]
    if eight:
        m8, v8 = _check_moments8(exp_avgs, counts, index, "exp_avgs"), _check_moments8(exp_avg_sqs, counts, index, "exp_avg_sqs")
        cols += [[t.data_ptr() for t in ts] for ts in (m8[0], v8[0], m8[1], v8[1])]
    else:
        if any([isinstance(m, Moment8) for m in (*exp_avgs, *exp_avg_sqs)]):
            raise ValueError("float32 moments expected beside float32 moments")
        _check(exp_avgs, torch.float32, index, shapes, "exp_avgs")
        _check(exp_avg_sqs, torch.float32, index, shapes, "exp_avg_sqs")
        cols += [[t.data_ptr() for t in exp_avgs], [t.data_ptr() for t in exp_avg_sqs], zeros, zeros]
    if masters is not None:
        _check(masters, torch.float32, index, shapes, "masters")
    cols += [zeros if masters is None else [w.data_ptr() for w in masters], counts]
    written = [a for f in (0, 2, 3, 4, 5) for a, c in zip(cols[f], counts) if c and a]
    written += [a for a, p, c in zip(cols[6], cols[0], counts) if c and a and a != p]
    if len(set(written)) != len(written):
        raise ValueError("a parameter, moment or master is listed twice")
    count = None
    if isinstance(dither, torch.Tensor):
        _check([dither], torch.int64, index, [1], "dither")
        count, dither = dither.data_ptr(), 0
    elif dither is None:
        dither = 0
    elif int(dither) != dither or dither < 1:
        raise ValueError(f"dither {dither}: the number of this step, from 1")
    on_device(first)
    if factors is None:
        if step is None or int(step) != step or step < 1:
            raise ValueError(f"step {step}: the number of this step, from 1, or `factors`")
        if torch.cuda.is_current_stream_capturing():
            raise _lib.CafeError("a captured step would repeat the same step number: use adamw_tick and `factors`")
        step = int(step)
    else:
        _check([factors], torch.float32, index, [3], "factors")
        step = 0
    if eight and dither and torch.cuda.is_current_stream_capturing():
        raise _lib.CafeError("a captured step would repeat the same random bits: give `dither` as a tensor")
    flat = (ctypes.c_int64 * (8 * n))(*[a for c in cols for a in c])
    with launch_on(first) as st:
        _lib.check(_lib.load().cafe_adamw_dither_dev(flat, n, DTYPE_CODE[dtype], 8 if eight else 32, float(lr), float(betas[0]),
                                                     float(betas[1]), float(eps), float(weight_decay), step,
                                                     None if factors is None else factors.data_ptr(), int(dither), count, st),
                   "cafe_adamw_dither_dev")
    torch.autograd.graph.increment_version([p for p in params if not p.is_inference()])     # a backward that kept one says so


def adamw_tick(step, factors, *, lr, betas=(0.9, 0.999), weight_decay=0.01):
    """step (an int64 tensor of one on the device) += 1, and `factors` (float32, three) for that step of adamw_step.  lr: a
    number, or a float32 tensor of one on the same device that is read when the launch runs.  May be captured."""
    if step.dtype is not torch.int64 or step.numel() != 1 or factors.device != step.device:
        raise ValueError("step: an int64 tensor of one element, on the device of `factors`")
    _check([factors], torch.float32, step.get_device(), [3], "factors")
    ptr = None
    if isinstance(lr, torch.Tensor):
        if lr.dtype is not torch.float32 or lr.numel() != 1 or lr.device != step.device:
            raise ValueError("lr: a number or a float32 tensor of one element on the device of `step`")
        ptr, lr = lr.data_ptr(), 0.0
    on_device(step)
    with launch_on(step) as st:
        _lib.check(_lib.load().cafe_adamw_tick_dev(step.data_ptr(), ptr, float(lr), float(betas[0]), float(betas[1]),
                                                   float(weight_decay), factors.data_ptr(), st), "cafe_adamw_tick_dev")


def moment8_values(exp_avgs, exp_avg_sqs):
    """The float32 values (1-d tensors) that two lists of Moment8 stand for, first moments and second moments, in one launch."""
    both = [*exp_avgs, *exp_avg_sqs]
    if not both:
        return [], []
    if not isinstance(both[0], Moment8):
        raise ValueError(f"Moment8 expected, not {type(both[0]).__name__}")
    first = both[0].codes
    counts = [m[0].numel() for m in both]
    codes, exponents = _check_moments8(both, counts, first.get_device(), "moments")
    on_device(first)
    sizes = [v for n in counts for v in (n, -n & 3)]             # slices of one array, on boundaries of 16 bytes
    out = torch.empty(sum(sizes), dtype=torch.float32, device=first.device).split(sizes)[::2]
    cols = ([t.data_ptr() for t in codes], [t.data_ptr() for t in exponents], [t.data_ptr() for t in out], counts,
            [0] * len(exp_avgs) + [1] * len(exp_avg_sqs))
    table = (ctypes.c_int64 * (5 * len(both)))(*[a for c in cols for a in c])
    with launch_on(first) as st:
        _lib.check(_lib.load().cafe_moment8_values_dev(table, len(both), st), "cafe_moment8_values_dev")
    return list(out[:len(exp_avgs)]), list(out[len(exp_avgs):])


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update in one launch per type and step count.

    state_bits: 32, or 8 for moments of one byte per value (plus one per 256): right on average, each within some 20 % (their
    rounding is random, by a hash that repeats from run to run).  master_weights: bfloat16 and float16
    parameters keep a float32 copy that the steps accumulate in (default True; ignored for float32).  capturable: the
    step count of a parameter group lives on the device, so that step() can be captured into a graph and replayed; lr may
    then be a float32 tensor of one element on the device, and parameters without a gradient are skipped but do not lag
    behind the group's count.  Parameters are contiguous; sparse gradients are refused.  Master weights are what is stepped:
    whoever writes 16-bit parameters in between (a checkpoint) clears `state` or loads the state that belongs to them."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32, master_weights=True,
                 capturable=False):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits {state_bits}: 8 or 32")
        if isinstance(lr, torch.Tensor) and not capturable:
            raise ValueError("lr as a tensor needs capturable=True")
        for name, v, ok in (("lr", lr, isinstance(lr, torch.Tensor) or lr >= 0), ("eps", eps, eps >= 0),
                            ("weight_decay", weight_decay, weight_decay >= 0),
                            ("betas", betas, all(0 <= b < 1 for b in betas) and len(betas) == 2)):
            if not ok:
                raise ValueError(f"{name} {v}")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=master_weights, capturable=capturable))

    def _init_state(self, p, group):
        if p.is_cuda and torch.cuda.is_current_stream_capturing():
            raise _lib.CafeError("run one step with this parameter's gradient before the capture: replays would clear its moments")
        st = self.state[p]
        st["step"] = 0
        if group["state_bits"] == 8:
            for name in ("exp_avg", "exp_avg_sq"):
                st[name + "_codes"], st[name + "_exponents"] = Moment8.zeros(p.numel(), p.device)
        else:
            st["exp_avg"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            st["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        if group["master_weights"] and p.dtype is not torch.float32:
            st["master"] = p.detach().float().clone(memory_format=torch.contiguous_format)
        return st

    @staticmethod
    def _moments(st):
        if "exp_avg_codes" in st:
            return Moment8(st["exp_avg_codes"], st["exp_avg_exponents"]), Moment8(st["exp_avg_sq_codes"], st["exp_avg_sq_exponents"])
        return st["exp_avg"], st["exp_avg_sq"]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            sets = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.layout is not torch.strided:
                    raise ValueError("sparse gradients are not supported: the sketch-backed tables have their own update")
                st = self.state[p] if self.state.get(p) else self._init_state(p, group)
                if not group["capturable"]:
                    st["step"] += 1
                key = (p.device, p.dtype, st["step"], "exp_avg_codes" in st, "master" in st)
                sets.setdefault(key, []).append((p, st))
            ticked = {}
            for (device, _, step, _, master), members in sets.items():
                kw = dict(lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"], step=step, dither=step)
                if group["capturable"]:
                    if device not in ticked:
                        ticked[device] = self._tick(group, device)
                    kw.update(step=None, lr=0.0, factors=ticked[device][1], dither=ticked[device][0])
                moments = [self._moments(st) for _, st in members]
                adamw_step([p for p, _ in members], [p.grad for p, _ in members], [m for m, _ in moments], [v for _, v in moments],
                           masters=[st["master"] for _, st in members] if master else None, **kw)
        return loss

    @staticmethod
    def _tick(group, device):
        """(count, factors): the group's device-side step count on `device`, advanced, and its factors."""
        counts = group.setdefault("device_step", {})
        key = str(device)
        if key not in counts:
            if torch.cuda.is_current_stream_capturing():
                raise _lib.CafeError("run one step before the capture: it creates the device-side step count")
            counts[key] = (torch.zeros(1, dtype=torch.int64, device=device), torch.empty(3, dtype=torch.float32, device=device))
        count, factors = counts[key]
        adamw_tick(count, factors, lr=group["lr"], betas=group["betas"], weight_decay=group["weight_decay"])
        return count, factors

    def state_dict(self):
        out = super().state_dict()
        for group in out["param_groups"]:
            if "device_step" in group:
                group["device_step"] = {k: int(c) for k, (c, _) in group["device_step"].items()}
        return out

    def load_state_dict(self, state_dict):
        """torch's, except that moments, codes and master weights keep their own types (torch casts floating state to the
        parameter's).  Another optimizer's state is refused."""
        for g in state_dict["param_groups"]:
            if not self.defaults.keys() <= g.keys():
                raise ValueError(f"not a state of this optimizer: no {sorted(self.defaults.keys() - g.keys())}")
        super().load_state_dict(state_dict)
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        mine = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(saved, mine):
            if i in state_dict["state"]:
                self.state[p] = {k: v.detach().to(p.device).clone() if isinstance(v, torch.Tensor) else v
                                 for k, v in state_dict["state"][i].items()}
        for group in self.param_groups:
            counts = group.pop("device_step", None)
            if counts:                          # resumed on another device: the count is the group's
                devices = {p.device for p in group["params"]}
                group["device_step"] = {str(d): (torch.full((1,), int(counts.get(str(d), max(counts.values()))), dtype=torch.int64, device=d),
                                                 torch.empty(3, dtype=torch.float32, device=d)) for d in devices}
