"""Linear layers with their bias, activation and residual in one launch, and their gradients.

The heads of the reference's models are stacks of these (dlrm_s_pytorch.py:213-251 create_mlp; wdl.py:704-721 adds the
wide part's logit to the deep part's last activation).  Here a layer is

    y = act(x W^T + b) + residual           dz = dy * act'(z),  dx = dz W,  dW = dz^T x,  db = column sums of dz

on the matrix units (cafe_amd/csrc/cafe_linear.hip), float32, bfloat16 or float16, sums in float32.  `linear` is
differentiable; `linear_forward` / `linear_backward` are the same two passes for a training step that is written out;
`run_mlp` sends an nn.Sequential of Linear and activation modules through `linear`."""
from functools import lru_cache
from typing import NamedTuple

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

DTYPE_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {"none": 0, "relu": 1, "sigmoid": 2, "gelu": 3, "silu": 4}
_SLOPE = 5


class Slope(NamedTuple):
    """What a forward keeps for its backward: the activation's slopes act'(z), float32 whatever x's type."""
    values: torch.Tensor


def on_device(t):
    """Raises unless `t` lives on a GPU (there is no CPU path)."""
    if not t.is_cuda:
        raise _lib.CafeError("cafe_amd needs GPU tensors: there is no CPU path in this package")


def differentiated(*tensors):
    """Whether a call on `tensors` (or None) goes through its autograd function: one requires grad, or a level of forward-mode
    differentiation is open.  There one may carry a tangent, without requiring grad; the function raises for it."""
    return (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)) or forward_ad._current_level >= 0


class launch_on:
    """The current stream of `t`'s device, with that device current inside the block."""
    __slots__ = ("index", "before")

    def __init__(self, t):
        self.index = t.device.index

    def __enter__(self):
        self.before = torch._C._cuda_getDevice()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


@lru_cache(maxsize=4096)
def _fwd_ws(m, k, n, code):
    return _lib.load().cafe_linear_fwd_ws(m, k, n, code)


@lru_cache(maxsize=4096)
def _bwd_ws(m, k, n, code, act):
    return _lib.load().cafe_linear_bwd_ws(m, k, n, code, act)


def _rows(t):
    """`t` as rows whose elements are adjacent, and the stride between rows (a view wherever one exists)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.shape[1] > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0)


def _check(x, weight, bias, activation, residual):
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation {activation!r}: one of {sorted(ACTIVATIONS)}")
    if x.dtype not in DTYPE_CODE:
        raise ValueError(f"float32, bfloat16 or float16 expected, not {x.dtype}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} does not fit weight {tuple(weight.shape)} ([out, in])")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError(f"bias {tuple(bias.shape)} does not fit weight {tuple(weight.shape)}")
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise ValueError(f"{name} is {t.dtype} on {t.device}, x is {x.dtype} on {x.device}")
    on_device(x)


def _forward(x, weight, bias, act, residual, keep):
    """x [M, K], residual [M, N] or None.  Returns (y, kept): the activation's slopes; y itself for relu without a
    residual; None without an activation or where not asked for."""
    L = _lib.load()
    x, ldx = _rows(x)
    weight, ldw = _rows(weight)
    m, k, n = x.shape[0], x.shape[1], weight.shape[0]
    code = DTYPE_CODE[x.dtype]
    y = torch.empty(m, n, dtype=x.dtype, device=x.device)
    kept, ldr, rp = None, 0, None
    if residual is not None:
        residual, ldr = _rows(residual)
        rp = residual.data_ptr()
    if bias is not None:
        bias = bias.contiguous()
    if keep and act:
        if act == ACTIVATIONS["relu"] and residual is None:
            kept = y
        else:
            kept = torch.empty(m, n, dtype=torch.float32, device=x.device)
    with launch_on(x) as st:
        need = _fwd_ws(m, k, n, code)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need > 0 else None
        _lib.check(L.cafe_linear_fwd_dev(x.data_ptr(), ldx, weight.data_ptr(), ldw, None if bias is None else bias.data_ptr(),
                                         rp, ldr, y.data_ptr(), n, None if kept is None or kept is y else kept.data_ptr(), n,
                                         m, k, n, code, act, None if ws is None else ws.data_ptr(), need, st),
                   "cafe_linear_fwd_dev")
    return y, kept


def _backward(grad, x, weight, kept, act, need):
    """act: the code that says what `kept` holds (include/cafe_hip.h, cafe_linear_bwd_dev)."""
    L = _lib.load()
    grad, ldg = _rows(grad)
    x, ldx = _rows(x)
    weight, ldw = _rows(weight)
    m, k, n = x.shape[0], x.shape[1], weight.shape[0]
    code = DTYPE_CODE[x.dtype]
    ldk, kp = 0, None
    if act:
        kept, ldk = _rows(kept)
        kp = kept.data_ptr()
    new = lambda *shape: torch.empty(shape, dtype=x.dtype, device=x.device)            # noqa: E731
    dx = new(m, k) if need[0] else None
    dw = new(n, k) if need[1] else None
    db = new(n) if need[2] else None
    with launch_on(x) as st:
        size = _bwd_ws(m, k, n, code, act)
        ws = torch.empty(size, dtype=torch.uint8, device=x.device) if size > 0 else None
        p = lambda t: None if t is None else t.data_ptr()                              # noqa: E731
        _lib.check(L.cafe_linear_bwd_dev(grad.data_ptr(), ldg, x.data_ptr(), ldx, weight.data_ptr(), ldw, kp, ldk, p(dx), k,
                                         p(dw), p(db), m, k, n, code, act, p(ws), size, st), "cafe_linear_bwd_dev")
    return dx, dw, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        y, kept = _forward(x, weight, bias, act, residual, any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, weight, kept)
        ctx.act, ctx.has_res = act if kept is None or kept is y else _SLOPE, residual is not None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if any(need[:3]):
            dx, dw, db = _backward(grad, x, weight, kept, ctx.act, need[:3])
        return dx, dw, db, grad if ctx.has_res and need[3] else None, None


def linear(x, weight, bias=None, activation="none", residual=None):
    """act(x weight^T + bias) + residual.

    x: [..., K] and weight: [N, K] (an nn.Linear's), bias: [N] or None, residual: anything that broadcasts to [..., N];
    all float32, bfloat16 or float16, on one GPU.  activation: "none", "relu", "sigmoid", "gelu" (z Phi(z)) or "silu".
    Rows may be strided views.  Runs on the current stream of x's device.  Differentiable once in x, weight, bias and
    residual, not in forward mode; the backward keeps x, weight and, for every activation but relu without a residual, one more [..., N]
    tensor, the activation's slopes in float32."""
    _check(x, weight, bias, activation, residual)
    lead = x.shape[:-1]
    n = weight.shape[0]
    if residual is not None:
        residual = residual.expand(*lead, n).reshape(-1, n) if x.dim() != 2 or residual.shape != (lead[0], n) else residual
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1]) if x.shape[-1] else x.new_empty(lead.numel(), 0)
    act = ACTIVATIONS[activation]
    if differentiated(x, weight, bias, residual):
        y = _Linear.apply(x2, weight, bias, residual, act)
    else:
        y = _forward(x2, weight, bias, act, residual, False)[0]
    return y if x.dim() == 2 else y.view(*lead, n)


def linear_forward(x, weight, bias=None, activation="none", residual=None):
    """`linear` without autograd for x [M, K]: (y, kept), kept being what linear_backward asks for (None for "none";
    y itself for "relu" without a residual; else a Slope)."""
    _check(x, weight, bias, activation, residual)
    if x.dim() != 2:
        raise ValueError(f"x [M, K] expected, not {tuple(x.shape)}")
    if residual is not None and residual.shape != (x.shape[0], weight.shape[0]):
        raise ValueError(f"residual {tuple(residual.shape)}, the output is {(x.shape[0], weight.shape[0])}")
    with torch.no_grad():
        y, kept = _forward(x, weight, bias, ACTIVATIONS[activation], residual, True)
    return y, kept if kept is None or kept is y else Slope(kept)


def linear_backward(grad, x, weight, kept=None, activation="none", need=(True, True, True)):
    """(dx, dweight, dbias) for the gradient of the output, grad [M, N]; None in the place of what `need` declines.
    kept: as linear_forward returned it, or a tensor [M, N] of the values before the activation (for "relu" any tensor
    of their sign)."""
    _check(x, weight, None, activation, grad)
    shape = (x.shape[0], weight.shape[0])
    if x.dim() != 2 or tuple(grad.shape) != shape:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} do not fit grad {tuple(grad.shape)}")
    act = ACTIVATIONS[activation]
    want = x.dtype
    if isinstance(kept, Slope):
        kept, act, want = kept.values, _SLOPE, torch.float32
    if act:
        if kept is None or tuple(kept.shape) != shape or kept.dtype != want or kept.device != x.device:
            raise ValueError(f"activation {activation!r} needs what its forward kept: a Slope (float32), or the values before the "
                             f"activation in x's type, of shape {shape} on x's device")
    with torch.no_grad():
        return _backward(grad, x, weight, kept, act, tuple(need))


def _plain(modules):
    """Raises unless calling each is its class's forward and nothing else: run_mlp goes by what the class stands for."""
    anywhere = nn.modules.module._has_any_global_hook()
    for m in modules:
        if not isinstance(m, nn.Module):
            raise ValueError(f"modules expected, not {type(m).__name__}")
        own = m.__dict__
        if anywhere or own["_forward_hooks"] or own["_forward_pre_hooks"] or own["_backward_hooks"] or own["_backward_pre_hooks"]:
            raise ValueError(f"{type(m).__name__} with hooks (weight_norm registers one): run_mlp would pass them by")
        if "forward" in own:
            raise ValueError(f"{type(m).__name__} with a forward of its own: run_mlp would pass it by")
    return modules


_ACTIVATION_OF = {nn.ReLU: "relu", nn.Sigmoid: "sigmoid", nn.SiLU: "silu", nn.Identity: "none"}


def mlp_modules(layers):
    """The modules of an nn.Sequential or a list, as run_mlp takes them; refuses what it refuses of the container."""
    if isinstance(layers, nn.Module):
        if type(layers) is not nn.Sequential:
            raise ValueError(f"nn.Sequential or a list of modules expected, not {type(layers).__name__}")
        _plain([layers])
        return _plain(list(layers._modules.values()))
    return _plain(list(layers))


def run_mlp(layers, x, residual=None):
    """An nn.Sequential of nn.Linear layers, each followed by its activation module or by the next Linear, one launch per
    layer; `residual` is added to the last layer's output.  `layers` may be a list of such modules.  What their classes do is
    done, so modules whose call does something else are refused: subclasses (a parametrized Linear is one), hooks."""
    mods = mlp_modules(layers)
    at = 0
    while at < len(mods):
        lin = mods[at]
        if type(lin) is not nn.Linear:
            raise ValueError(f"nn.Linear itself expected at {at}, not {type(lin).__name__}")
        act, step = "none", 1
        if at + 1 < len(mods) and not isinstance(mods[at + 1], nn.Linear):
            nxt = mods[at + 1]
            exact_gelu = type(nxt) is nn.GELU and nxt.approximate == "none"
            act = "gelu" if exact_gelu else _ACTIVATION_OF.get(type(nxt))
            if act is None:
                raise ValueError(f"activation module {nxt} has no fused form")
            step = 2
        at += step
        x = linear(x, lin.weight, lin.bias, act, residual if at >= len(mods) else None)
    return x
