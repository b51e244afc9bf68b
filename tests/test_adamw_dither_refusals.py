"""cafe_amd.adamw refuses step numbers that it cannot round by, before anything is launched (no GPU needed)."""
import ctypes

import pytest
import torch

from cafe_amd import _lib
from cafe_amd.adamw import Moment8, adamw_step


@pytest.mark.parametrize("dither", [0, -1, 1.5, torch.zeros(1), torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int32)])
def test_numbers(dither):
    z = lambda: torch.zeros(5)                                                         # noqa: E731
    m = lambda: Moment8.zeros(5, "cpu")                                                # noqa: E731
    with pytest.raises(ValueError, match="dither"):
        adamw_step([z()], [z()], [m()], [m()], step=1, lr=0.1, dither=dither)


def test_c_entry_point():
    L = _lib.load()
    table = (ctypes.c_int64 * 8)(4096, 4096, 4096, 4096, 4096, 4096, 0, 0)             # no values: nothing to do
    call = lambda d: L.cafe_adamw_dither_dev(table, 1, 0, 8, 0.1, 0.9, 0.99, 0.0, 0.0, 1, None, d, None, None)   # noqa: E731
    assert call(0) == 0 and call(9) == 0 and call(1 << 40) == 0
    assert call(-1) != 0 and b"dither" in L.cafe_last_error()
