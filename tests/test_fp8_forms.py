"""The rules that choose a kernel (csrc/fp8_layout.h, compiled for the CPU) against the forms that the GPU tests name."""
import ctypes as C

import pytest

from tests import fp8_forms as K
from tests.test_fp8_layout import _choose, _pair, rules


def form(m, n, k, groups=1, grouped=False, exact=False):
    tile, rows, parts = _choose(m, n, k, groups, grouped, exact)
    if tile:
        return tile, parts
    L = rules()
    L.row_share.argtypes = [C.c_uint64, C.c_uint32, C.c_uint32, C.c_void_p]
    tiles = L.row_tiles(m, groups, rows)
    if rows == 16:
        return (rows,) + _pair(L.row_share, tiles, n, k)
    return rows, 2, 8 if tiles * -(-n // 32) < 256 else 4


def held(want, exact):
    """The form of outputs that need sums of f32: tiles of 128 at most."""
    return (128,) + want[1:] if exact and want[0] == 256 else want


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("size,want", K.CUT_TILES)
def test_cut_tiles(size, want, exact):
    assert form(*size, exact=exact) == held(want, exact)
