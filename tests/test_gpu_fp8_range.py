"""Operators of 8-bit floating-point codes on the GPU at the ends of their range, against the plain 64-bit forms of tests/fp8_ref.py."""
import numpy as np
import pytest

from tests import fp8_ref as R
from tests.test_gpu_fp8 import F, _held, _quantize  # noqa: F401 (F is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_quantize_gates_far_below_zero(F, dtype):
    """Gates around -87 to -89, where 1 + exp(-gate) reaches f32's end, and below, where exp(gate) alone is no f32 any more while
    its product with a large value is. The bounds of test_quantize_gated, whose error of 2^-20 covers four exponentials of 2^-23
    and eight roundings of 2^-24, and half of f32's smallest step for x that is subnormal."""
    near = np.linspace(-89.5, -86.0, 128 * 8)
    far = np.concatenate([np.linspace(top, top - 1.5, 128) for top in (-80, -100, -110, -130, -150, -172, -176, -188)])
    k = near.size + far.size
    values = [1.0, -3.0, 1000.0, 60000.0] + ([] if dtype == "f16" else [1e30, -3e38])
    x = np.concatenate([np.repeat(np.array(values)[:, None], k, 1), np.repeat(np.concatenate([near, far])[None], len(values), 0)], 1)
    x = _held(x, dtype)
    codes, scales = _quantize(F, x, dtype, gated=True)
    y = R.gated(x)
    want = R.quantize(y)[1].astype(np.float64)
    assert (np.abs(scales - want) <= 2.0 ** -20 * want).all()
    s = R.spread(scales.astype(np.float64), k)
    v = R.VALUES[codes] * s
    step = np.maximum(2.0 ** np.floor(np.log2(np.maximum(np.abs(y) / s, 2.0 ** -6))), 2.0 ** -6) / 8
    assert (np.abs(v - y) <= s * step / 2 * (1 + 2.0 ** -18) + 2.0 ** -19 * np.abs(y) + 2.0 ** -149).all()
    assert (R.VALUES[codes[-1]] != 0).any()


def test_quantize_gates_without_end(F):
    """The lowest gates give zeros, minus infinity spoils its block only."""
    x = np.ones((4, 512))
    x[0, 256:], x[1, 256:], x[2, 256:] = -3.4e38, -1e5, -400.0
    x[2, :256] = 3e38
    x[3, 300] = -np.inf
    codes, scales = _quantize(F, x.astype(np.float32).astype(np.float64), "f32", gated=True)
    assert (R.VALUES[codes[:3]] == 0).all() and (scales[:3] == np.float32(R.SMALLEST_SCALE)).all()
    assert np.isnan(scales[3]).tolist() == [True, False] and (codes[3, :128] == 0).all()
