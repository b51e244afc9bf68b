"""cafe_amd.linear refuses what it has no kernel for before anything is launched (runs without a GPU)."""
import ctypes

import pytest
import torch
import torch.nn as nn

from cafe_amd import _lib
from cafe_amd.linear import linear, linear_backward, linear_forward, run_mlp

X, W, B = torch.zeros(3, 5), torch.zeros(7, 5), torch.zeros(7)


@pytest.mark.parametrize("args,kw", [
    ((X, W, B, "tanh"), {}),                                    # no such activation
    ((X.double(), W.double()), {}),                             # no such type
    ((X.half(), W), {}),                                        # mixed types
    ((X, W, B.bfloat16()), {}),
    ((torch.zeros(3, 6), W), {}),                               # widths
    ((X, W, torch.zeros(5)), {}),
    ((X, torch.zeros(7, 5, 1)), {}),
    ((torch.zeros(()), W), {}),
    ((X, W, B, "none", torch.zeros(3, 7).half()), {}),          # residual of another type
])
def test_arguments(args, kw):
    with pytest.raises(ValueError):
        linear(*args, **kw)


def test_no_cpu_path():
    with pytest.raises(_lib.CafeError):
        linear(X, W, B, "relu")
    with pytest.raises(_lib.CafeError):
        linear_forward(X, W)
    with pytest.raises(_lib.CafeError):
        linear_backward(torch.zeros(3, 7), X, W)
    with pytest.raises(_lib.CafeError):
        run_mlp(nn.Sequential(nn.Linear(5, 7), nn.ReLU()), X)


def test_mlp_layers():
    with pytest.raises(ValueError):
        run_mlp(nn.Sequential(nn.ReLU()), X)
    with pytest.raises(ValueError):
        run_mlp(nn.Sequential(nn.Linear(5, 7), nn.Tanh()), X)
    with pytest.raises(ValueError):
        run_mlp(nn.Sequential(nn.Linear(5, 7), nn.GELU(approximate="tanh")), X)


def test_c_entry_points():
    """Bad sizes, codes, strides, null pointers and short workspaces come back as errors, before any HIP call."""
    L = _lib.load()
    p = ctypes.c_void_p(4096)                                   # never read: every call below is refused
    for m, k, n, t in ((-1, 1, 1, 0), (1, -1, 1, 0), (1, 1, 1 << 31, 0), (1, 1, 1, 3), (1, 1, 1, -1)):
        assert L.cafe_linear_fwd_ws(m, k, n, t) == -1
        assert L.cafe_linear_bwd_ws(m, k, n, t, 0) == -1
    assert L.cafe_linear_bwd_ws(1, 1, 1, 0, 6) == -1 and L.cafe_linear_bwd_ws(1, 1, 1, 0, -1) == -1
    for t in range(3):                                          # every size that may be 0 has a workspace size
        for m in (0, 1, 70, 70000):
            for k in (0, 1, 5000):
                for n in (0, 1, 40):
                    assert L.cafe_linear_fwd_ws(m, k, n, t) >= 0 and L.cafe_linear_bwd_ws(m, k, n, t, 1) >= 0

    def fwd(x=p, ldx=5, w=p, ldw=5, res=None, ldr=0, y=p, ldy=7, kept=None, ldk=0, m=3, k=5, n=7, t=0, act=0, ws=None, size=1 << 40):
        return L.cafe_linear_fwd_dev(x, ldx, w, ldw, None, res, ldr, y, ldy, kept, ldk, m, k, n, t, act, ws, size, None)

    for kw in (dict(x=None), dict(w=None), dict(y=None), dict(ldy=6), dict(ldx=-1), dict(ldw=-5), dict(ldr=-1), dict(kept=p, ldk=6),
               dict(m=-1), dict(t=7), dict(act=5), dict(act=9), dict(m=64, k=1 << 20, n=64, ldx=1 << 20, ldw=1 << 20, ldy=64, size=-1)):
        assert fwd(**kw) != 0, kw
        assert L.cafe_last_error()
    assert fwd(m=0, x=None, w=None, y=None) == 0                # nothing to do

    def bwd(dy=p, lddy=7, x=p, w=p, kept=p, ldk=7, dx=p, lddx=5, dw=p, db=p, m=3, k=5, n=7, act=1, ws=p, size=1 << 40):
        return L.cafe_linear_bwd_dev(dy, lddy, x, 5, w, 5, kept, ldk, dx, lddx, dw, db, m, k, n, 0, act, ws, size, None)

    for kw in (dict(dy=None), dict(kept=None), dict(x=None), dict(w=None), dict(lddx=4), dict(lddy=-1), dict(ldk=-1), dict(size=0),
               dict(ws=None), dict(act=-1), dict(act=6), dict(k=-3)):
        assert bwd(**kw) != 0, kw
