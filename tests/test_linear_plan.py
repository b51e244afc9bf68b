"""Sizes that cafe_linear_plan and the workspaces refuse (no GPU needed)."""
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


def test_workspaces_that_no_number_holds():
    """2^31 - 1 squared, four bytes each: 2^64.  Refused with a message instead of a size that wrapped round."""
    L = _lib.load()
    big = (1 << 31) - 1
    for m, k, n in ((big, 1, big), (big, big, 1), (1, big, big)):
        for t in range(3):
            assert L.cafe_linear_fwd_ws(m, k, n, t) == -1 and b"2^48" in L.cafe_last_error()
            assert L.cafe_linear_bwd_ws(m, k, n, t, 2) == -1 and b"2^48" in L.cafe_last_error()
    assert L.cafe_linear_bwd_ws(1 << 24, 1, 1 << 24, 1, 2) >= 2 * 2 << 48                # the largest: two parts of two bytes
    p = ctypes.c_void_p(4096)                                   # never read
    assert L.cafe_linear_fwd_dev(p, 0, p, 1, None, None, 0, p, big, None, 0, big, 1, big, 0, 0, p, 1 << 62, None) != 0
    assert L.cafe_linear_bwd_dev(p, 0, p, 0, p, 0, p, 0, p, 1, p, p, big, 1, big, 0, 2, p, 1 << 62, None) != 0
