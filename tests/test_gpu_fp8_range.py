"""Operators of 8-bit floating-point codes on the GPU at the ends of their range, against the plain 64-bit forms of tests/fp8_ref.py."""
import numpy as np
import pytest
import torch

from tests import fp8_ref as R
from tests.test_gpu_fp8 import DT, F, _dev, _held, _ints, _near, _np, _padded, _quantize  # noqa: F401 (F is a fixture)

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


# ---------------------------------------------------------------- products

def _whole(r, m, n, k):
    """Codes of whole numbers with the scale 1: in each eight neighbours one product of 448 * 448, which the next eight take away,
    and seven of -2 .. 2. Sums of any of a block's are whole and below 2^24 and the blocks' sums are small, so that sums in f32 are
    exact in every order; the results stay below 2^11: exact in f16 too. (Products cut off below 2^-13 of a neighbour's would be
    gone.)"""
    a, b = np.ones((m, k)), r.integers(-2, 3, (n, k)).astype(np.float64)
    large = np.arange(0, k, 8)
    large = large[:large.size // 2 * 2]
    a[:, large] = 448.0
    b[:, large[0::2]], b[:, large[1::2]] = 448.0, -448.0
    return a, b


WHOLE = [(1, 300, 1024), (16, 96, 2048), (33, 96, 2048), (64, 1024, 8192), (300, 3000, 1160), (1500, 4100, 136), (2000, 4104, 512)]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("m,n,k", WHOLE)
def test_sums_are_f32(F, dtype, m, n, k):
    """Outputs of more bits than bf16's come from sums of f32, in every kernel."""
    a, b = _whole(np.random.default_rng(m), m, n, k)
    d = torch.full((m, n), 7.0, dtype=DT[dtype], device="cuda")
    x = [_padded(R.nearest(a)), torch.ones(m, R.blocks(k), device="cuda"), _padded(R.nearest(b)), torch.ones(R.blocks(n), R.blocks(k), device="cuda")]
    F.Fp8Matmul(*x, d).encode()
    torch.cuda.synchronize()
    assert np.array_equal(_np(d), a @ b.T)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("sizes,n,k", [([1, 2, 0, 9], 100, 1024), ([40, 7, 200], 1536, 272), ([900, 0, 1030, 513], 4100, 136)])
def test_grouped_sums_are_f32(F, dtype, sizes, n, k):
    r = np.random.default_rng(n)
    m, experts = sum(sizes), len(sizes)
    a, _ = _whole(r, m, 1, k)
    b = np.stack([_whole(r, 1, n, k)[1] for _ in sizes])
    start = np.concatenate([[0], np.cumsum(sizes)])
    d = torch.full((m, n), 7.0, dtype=DT[dtype], device="cuda")
    x = [_padded(R.nearest(a)), torch.ones(m, R.blocks(k), device="cuda"), _padded(R.nearest(b)),
         torch.ones(experts, R.blocks(n), R.blocks(k), device="cuda")]
    F.Fp8GroupedMatmul(*x, d, _ints(start)).encode()
    torch.cuda.synchronize()
    assert np.array_equal(_np(d), np.concatenate([a[start[e]:start[e + 1]] @ b[e].T for e in range(experts)]))


def test_more_workgroups_than_a_launch_holds(F):
    """2^22 rows, N 4096, K 64: 2^24 workgroups of 256 threads, in two launches. Rows on both sides of where the second one
    begins (the last row tile), and no row left out."""
    m, n, k = 2 ** 22, 4096, 64
    r = np.random.default_rng(5)
    a = torch.randint(0, 0x7f, (m, k), dtype=torch.uint8, device="cuda")
    sa = torch.rand(m, 1, device="cuda") + 0.5
    b, sb = R.nearest(r.normal(0, 110, (n, k))), r.random((32, 1)).astype(np.float32)
    d = torch.full((m, n), 7.0, dtype=torch.bfloat16, device="cuda")
    F.Fp8Matmul(a, sa, _padded(b), _dev(sb), d).encode()
    torch.cuda.synchronize()
    assert not any((part == 7).all(1).any() for part in d.split(m // 16))
    at = torch.tensor([0, 1, 2 ** 21, m - 65, m - 33, m - 32, m - 31, m - 1], device="cuda")
    want, mag, cut = R.product(a[at].cpu().numpy(), sa[at].cpu().numpy(), b, sb)
    _near(_np(d[at]), want, R.bound(want, mag, cut, k, "bf16"), "bf16")


def test_sizes_past_32_bits_are_refused(F, qmm):
    """One row seen 2^32 + 1 times is no call of one row."""
    many = 2 ** 32 + 1
    codes, scales = F.new_rows(1, 16)
    row = torch.zeros(1, 16, device="cuda")
    for call in (lambda: F.Fp8Quantize(row.expand(many, 16), codes.expand(many, 16), scales.expand(many, 1)),
                 lambda: F.Fp8Matmul(codes, scales, codes.expand(many, 16), scales.expand(many // 128 + 1, 1), torch.zeros(1, 1, device="cuda").expand(1, many)),
                 lambda: F.Fp8Matmul(codes.expand(many, 16), scales.expand(many, 1), codes, scales, torch.zeros(1, 1, device="cuda").expand(many, 1)),
                 lambda: F.Fp8GroupedMatmul(codes.expand(many, 16), scales.expand(many, 1), codes[None], scales[None],
                                            torch.zeros(1, 1, device="cuda"), _ints([0, 1]), a_rows=_ints([0])),
                 lambda: F.ExpertPlan(_ints([[0]]), 1, 2 ** 32),
                 lambda: F.ExpertPlan(_ints([[0]]), 2 ** 32 + 1)):
        with pytest.raises(qmm.MatmulError) as e:
            call()
        assert e.value.status == qmm.INVALID_ARGUMENT
