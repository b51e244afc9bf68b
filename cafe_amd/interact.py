"""DLRM's dot interaction as one launch in each direction (cafe_amd/csrc/cafe_interact.hip).

The reference concatenates the rows, multiplies them with torch.bmm, picks the pairs below the diagonal by index and
concatenates again (dlrm_s_pytorch.py:779-809).  `dot_interaction` reads the embedding rows as the collection wrote them,
[F, B, D] float32, beside dense rows of the head's own type, and writes what the top MLP reads."""
import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .linear import DTYPE_CODE, differentiated, launch_on, on_device

MAX_FEATURES = 128


def _adjacent(t):
    return t if t is None or t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _forward(x, emb, itself, dtype):
    f, b, d = emb.shape
    nf = f + (x is not None)
    width = (nf * (nf + 1) if itself else nf * (nf - 1)) // 2 + (d if x is not None else 0)
    x, emb = _adjacent(x), _adjacent(emb)
    out = torch.empty(b, width, dtype=dtype, device=emb.device)
    if b == 0 or d == 0:                        # empty rows: every product is 0
        return out.zero_()
    with launch_on(emb) as st:
        _lib.check(_lib.load().cafe_interact_fwd_dev(None if x is None else x.data_ptr(), 0 if x is None else x.stride(0),
                                                     emb.data_ptr(), emb.stride(0), emb.stride(1), b, f, d, int(itself),
                                                     DTYPE_CODE[emb.dtype], DTYPE_CODE[dtype], out.data_ptr(), width, st),
                   "cafe_interact_fwd_dev")
    return out


class _Interact(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, emb, itself, dtype):
        ctx.save_for_backward(x, emb)
        ctx.itself = itself
        return _forward(x, emb, itself, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, emb = ctx.saved_tensors
        f, b, d = emb.shape
        want_x, want_e = ctx.needs_input_grad[:2]
        grad = _adjacent(grad)
        xa, ea = _adjacent(x), _adjacent(emb)
        dx = torch.empty(b, d, dtype=x.dtype, device=x.device) if want_x else None
        de = torch.empty(f, b, d, dtype=emb.dtype, device=emb.device) if want_e else None
        if b == 0 or d == 0:
            return dx, de, None, None
        with launch_on(emb) as st:
            _lib.check(_lib.load().cafe_interact_bwd_dev(
                grad.data_ptr(), grad.stride(0), None if xa is None else xa.data_ptr(), 0 if xa is None else xa.stride(0),
                ea.data_ptr(), ea.stride(0), ea.stride(1), b, f, d, int(ctx.itself), DTYPE_CODE[emb.dtype], DTYPE_CODE[grad.dtype],
                None if dx is None else dx.data_ptr(), d, None if de is None else de.data_ptr(), b * d, d, st), "cafe_interact_bwd_dev")
        return dx, de, None, None


def dot_interaction(x, emb, itself=False, dtype=None):
    """[x | <t_i, t_j> for j < i (j <= i with `itself`), i ascending] over the rows t = (x, emb[0], emb[1], ...) of every sample.

    x: [B, D] (the bottom MLP's output) or None; emb: [F, B, D].  The result is [B, (D +) pairs] of `dtype` (default: x's
    type, emb's without x).  x has the result's type; emb has it too or is float32.  At most 128 feature rows, x included.
    Products and sums are float32.  Rows may be strided views.  Runs on the current stream of emb's device;
    differentiable once in x and emb, not in forward mode."""
    if emb.dim() != 3:
        raise ValueError(f"emb [fields, batch, dim] expected, not {tuple(emb.shape)}")
    dtype = (emb.dtype if x is None else x.dtype) if dtype is None else dtype
    if dtype not in DTYPE_CODE or emb.dtype not in (torch.float32, dtype):
        raise ValueError(f"embedding rows are float32 or of the result's type: {emb.dtype} and {dtype}")
    if x is not None and (x.shape != emb.shape[1:] or x.dtype != dtype or x.device != emb.device):
        raise ValueError(f"x {tuple(x.shape)} {x.dtype} on {x.device} does not fit emb {tuple(emb.shape)} on {emb.device}, result {dtype}")
    nf = emb.shape[0] + (x is not None)
    if not 1 <= nf <= MAX_FEATURES:
        raise ValueError(f"{nf} feature rows: 1 .. {MAX_FEATURES} expected")
    on_device(emb)
    if differentiated(x, emb):
        return _Interact.apply(x, emb, bool(itself), dtype)
    return _forward(x, emb, bool(itself), dtype)
