"""Every tile that the products of a layer are cut into, in every operand layout: whole tiles and ragged edges, the reduction in
one piece and in slices, long enough for the inner loops (ten and more steps of 128 bytes per slice).

The sizes are found from the estimate that chooses the tile; the test asks the library which tile it takes, so that sizes
that no longer reach theirs fail here.  Tolerances: as in test_gpu_linear.py, and for dz in two parts as in
test_gpu_linear_gradients.py."""
import ctypes

import pytest
import torch

from cafe_amd import _lib
from cafe_amd.linear import ACTIVATIONS, DTYPE_CODE, linear_backward, linear_forward
from test_gpu_linear import check_backward, check_forward, make
from test_gpu_linear_gradients import rounded_once

PRODUCTS = ("forward", "dx", "dw")
# type, product, rows and columns of the tile, slices, parts of dz, (m, k, n); sizes one above and one below take the same
TILES = [
    ("float32", "forward", 64, 64, False, 1, (544, 640, 1184)),
    ("float32", "forward", 64, 64, True, 1, (672, 640, 480)),
    ("float32", "forward", 64, 128, False, 1, (160, 640, 16512)),
    ("float32", "forward", 64, 128, True, 1, (160, 960, 5472)),
    ("float32", "forward", 128, 64, False, 1, (2208, 640, 1376)),
    ("float32", "forward", 128, 64, True, 1, (800, 960, 1248)),
    ("float32", "forward", 128, 128, False, 1, (1376, 640, 4448)),
    ("float32", "forward", 128, 128, True, 1, (1184, 1504, 1696)),
    ("float32", "dx", 64, 64, False, 1, (992, 672, 640)),
    ("float32", "dx", 64, 64, True, 1, (480, 672, 640)),
    ("float32", "dx", 64, 128, False, 1, (288, 10944, 640)),
    ("float32", "dx", 64, 128, True, 1, (160, 5600, 960)),
    ("float32", "dx", 128, 64, False, 1, (1952, 1568, 640)),
    ("float32", "dx", 128, 64, True, 1, (1248, 800, 960)),
    ("float32", "dx", 128, 128, False, 1, (3616, 1696, 640)),
    ("float32", "dx", 128, 128, True, 1, (1184, 1728, 1504)),
    ("float32", "dw", 64, 64, False, 1, (640, 1184, 544)),
    ("float32", "dw", 64, 64, True, 1, (640, 672, 480)),
    ("float32", "dw", 64, 128, False, 1, (640, 16640, 160)),
    ("float32", "dw", 64, 128, True, 1, (960, 5472, 160)),
    ("float32", "dw", 128, 64, False, 1, (640, 1376, 2208)),
    ("float32", "dw", 128, 64, True, 1, (960, 800, 1248)),
    ("float32", "dw", 128, 128, False, 1, (640, 4896, 1248)),
    ("float32", "dw", 128, 128, True, 1, (1312, 6592, 288)),
    ("16 bits", "forward", 64, 64, False, 1, (96, 640, 96)),
    ("16 bits", "forward", 64, 64, True, 1, (64, 10240, 64)),
    ("16 bits", "forward", 64, 128, False, 1, (160, 640, 8320)),
    ("16 bits", "forward", 64, 128, True, 1, (160, 2656, 2880)),
    ("16 bits", "forward", 128, 64, False, 1, (1184, 640, 864)),
    ("16 bits", "forward", 128, 64, True, 1, (608, 2816, 800)),
    ("16 bits", "forward", 128, 128, False, 1, (1184, 640, 1696)),
    ("16 bits", "forward", 128, 128, True, 1, (672, 5600, 480)),
    ("16 bits", "forward", 256, 128, False, 1, (1696, 640, 2432)),
    ("16 bits", "forward", 256, 128, True, 1, (160, 3232, 5504)),
    ("16 bits", "dx", 64, 64, False, 1, (64, 64, 640)),
    ("16 bits", "dx", 64, 64, False, 2, (64, 64, 640)),
    ("16 bits", "dx", 64, 64, True, 1, (64, 64, 10240)),
    ("16 bits", "dx", 64, 64, True, 2, (64, 64, 10240)),
    ("16 bits", "dx", 64, 128, False, 1, (160, 8224, 640)),
    ("16 bits", "dx", 64, 128, True, 1, (160, 2752, 2656)),
    ("16 bits", "dx", 64, 128, False, 2, (457, 2087, 641)),
    ("16 bits", "dx", 64, 128, True, 2, (77, 2691, 2087)),
    ("16 bits", "dx", 128, 64, False, 1, (800, 1248, 640)),
    ("16 bits", "dx", 128, 64, False, 2, (1184, 416, 640)),
    ("16 bits", "dx", 128, 64, True, 1, (672, 736, 2848)),
    ("16 bits", "dx", 128, 64, True, 2, (928, 160, 2720)),
    ("16 bits", "dx", 128, 128, False, 1, (2336, 864, 640)),
    ("16 bits", "dx", 128, 128, False, 2, (1824, 544, 640)),
    ("16 bits", "dx", 128, 128, True, 1, (672, 480, 5408)),
    ("16 bits", "dx", 128, 128, True, 2, (832, 608, 1920)),
    ("16 bits", "dx", 256, 128, False, 1, (1056, 3872, 640)),
    ("16 bits", "dx", 256, 128, False, 2, (1760, 1184, 640)),
    ("16 bits", "dx", 256, 128, True, 1, (160, 5472, 3232)),
    ("16 bits", "dx", 256, 128, True, 2, (2752, 160, 2560)),
    ("16 bits", "dw", 64, 64, False, 1, (640, 64, 64)),
    ("16 bits", "dw", 64, 64, False, 2, (640, 64, 64)),
    ("16 bits", "dw", 64, 64, True, 1, (10240, 64, 64)),
    ("16 bits", "dw", 64, 64, True, 2, (10240, 64, 64)),
    ("16 bits", "dw", 64, 128, False, 1, (640, 5472, 288)),
    ("16 bits", "dw", 64, 128, True, 1, (2656, 2784, 160)),
    ("16 bits", "dw", 64, 128, False, 2, (648, 2710, 324)),
    ("16 bits", "dw", 64, 128, True, 2, (2054, 2783, 75)),
    ("16 bits", "dw", 128, 64, False, 1, (640, 800, 1248)),
    ("16 bits", "dw", 128, 64, False, 2, (640, 608, 832)),
    ("16 bits", "dw", 128, 64, True, 1, (2816, 608, 800)),
    ("16 bits", "dw", 128, 64, True, 2, (2720, 160, 928)),
    ("16 bits", "dw", 128, 128, False, 1, (640, 1184, 1696)),
    ("16 bits", "dw", 128, 128, False, 2, (640, 736, 1376)),
    ("16 bits", "dw", 128, 128, True, 1, (5600, 672, 480)),
    ("16 bits", "dw", 128, 128, True, 2, (1920, 544, 928)),
    ("16 bits", "dw", 256, 128, False, 1, (640, 2400, 1696)),
    ("16 bits", "dw", 256, 128, False, 2, (640, 2400, 864)),
    ("16 bits", "dw", 256, 128, True, 1, (3232, 5472, 160)),
    ("16 bits", "dw", 256, 128, True, 2, (2560, 160, 2752)),
]
FOUND = {"float32": [torch.float32], "16 bits": [torch.bfloat16, torch.float16]}


def tile(t, product, act, m, k, n):
    out = (ctypes.c_int * 4)()
    _lib.check(_lib.load().cafe_linear_plan(m, k, n, DTYPE_CODE[t], ACTIVATIONS[act], PRODUCTS.index(product), out), "cafe_linear_plan")
    return tuple(out)


def test_every_tile_is_listed():
    """All tiles (256 x 128 in 16 bits only) x products x one or several slices x parts (dz in 16 bits: one and two)."""
    want = set()
    for kind, biggest in (("float32", []), ("16 bits", [(256, 128)])):
        for product in PRODUCTS:
            for bm, bn in biggest + [(128, 128), (128, 64), (64, 128), (64, 64)]:
                for parts in (1, 2) if kind == "16 bits" and product != "forward" else (1,):
                    want |= {(kind, product, bm, bn, sliced, parts) for sliced in (False, True)}
    assert want == {row[:6] for row in TILES}


@pytest.mark.parametrize("kind,product,bm,bn,sliced,parts,size", TILES)
def test_choice(kind, product, bm, bn, sliced, parts, size):
    for t in FOUND[kind]:
        for act in ("silu",) if parts == 2 else ("none", "relu"):
            for d in (0, 1, -1):
                got = tile(t, product, act, *(s + d for s in size))
                assert (got[0], got[1], got[2] > 1, got[3]) == (bm, bn, sliced, parts), (t, act, d)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,product,bm,bn,sliced,parts,size", TILES)
def test_tile(kind, product, bm, bn, sliced, parts, size):
    for t in FOUND[kind]:
        for d in (0, 1, -1):
            m, k, n = (s + d for s in size)
            if parts == 2:
                rounded_once(m, k, n, t, seed=m)
                continue
            for act in ("none", "relu"):
                x, w, b, r, dy = make(m, k, n, t, seed=m + k, residual=act == "none")
                if product == "forward":
                    y, kept = linear_forward(x, w, b, act, r)
                    check_forward(y, kept, x, w, b, r, act)
                else:
                    need = (product == "dx", product == "dw", product == "dw")
                    check_backward(linear_backward(dy, x, w, None if act == "none" else dy, act, need), dy, x, w, dy, act)
