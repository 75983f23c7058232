"""Products of 8-bit floating-point codes on the GPU in every kernel that takes them (tests/fp8_forms.py), against the plain 64-bit
forms of tests/fp8_ref.py."""
import numpy as np
import pytest
import torch

from tests import fp8_forms as K
from tests import fp8_ref as R
from tests.test_gpu_fp8 import DT, F, _dev, _near, _np, _operands, _padded  # noqa: F401 (F is a fixture)

pytestmark = pytest.mark.gpu


def _some(m, most=40):
    """Rows that are compared: at most some `most`, the first and the last of every 64 among them."""
    edges = np.concatenate([np.arange(0, m, 64), np.arange(63, m, 64), [m - 1]])
    return np.unique(np.concatenate([edges[:: max(1, len(edges) // (most // 2))], [0, m - 1], np.arange(0, m, max(1, m // (most // 2)))]))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("size,want", K.CUT_TILES)
def test_cut_column_tiles(F, dtype, size, want):
    """Column tiles whose first waves' columns are all there and whose last waves' are not; rows of d with a gap behind them."""
    m, n, k = size
    r = np.random.default_rng(m)
    a, sa, b, sb = _operands(r, m, n, k)
    full = torch.full((m, n + 8), 7.0, dtype=DT[dtype], device="cuda")
    F.Fp8Matmul(_padded(a), _dev(sa), _padded(b), _dev(sb), full[:, :n]).encode()
    torch.cuda.synchronize()
    assert (full[:, n:] == 7).all()
    at = _some(m)
    want, mag, cut = R.product(a[at], sa[at], b, sb)
    _near(_np(full[:, :n])[at], want, R.bound(want, mag, cut, k, dtype), dtype)
