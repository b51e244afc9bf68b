"""cafe_linear_plan refuses what it cannot answer (no GPU needed)."""
import ctypes

from cafe_amd import _lib


def test_c_entry_point():
    L = _lib.load()
    out = (ctypes.c_int * 4)()
    assert L.cafe_linear_plan(8192, 1024, 1024, 1, 4, 2, out) == 0 and out[3] == 2      # silu in bfloat16: dz in two parts
    assert L.cafe_linear_plan(8192, 1024, 1024, 0, 4, 2, out) == 0 and out[3] == 1
    assert L.cafe_linear_plan(1, 479, 1024, 1, 0, 0, out) == 0 and out[0] == 0          # one row: no tiles
    for bad in ((-1, 1, 1, 0, 0, 0), (1, 1, 1 << 31, 0, 0, 0), (1, 1, 1, 3, 0, 0), (1, 1, 1, 0, 6, 0), (1, 1, 1, 0, 0, 3), (1, 1, 1, 0, 0, -1)):
        assert L.cafe_linear_plan(*bad, out) != 0 and L.cafe_last_error()
    assert L.cafe_linear_plan(1, 1, 1, 0, 0, 0, None) != 0
