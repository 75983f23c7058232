"""Operators of 8-bit floating-point codes on the GPU against their plain 64-bit forms (tests/fp8_ref.py): codes, scales and
plans exactly, products and sums within the bounds derived there."""
import numpy as np
import pytest
import torch

from tests import fp8_ref as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module")
def F(qmm):
    from stark_amd import fp8
    return fp8


def _dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


def _ints(v):
    return torch.tensor(np.asarray(v, np.int64), dtype=torch.int32).cuda()


def _np(t):
    return t.detach().cpu().double().numpy() if t.is_floating_point() else t.cpu().numpy()


def _padded(codes):
    """Codes on the device, rows on 16-byte boundaries with NaN codes behind their ends."""
    k = codes.shape[-1]
    wide = -(-k // 16) * 16
    full = np.full(codes.shape[:-1] + (wide,), 0x7f, np.uint8)
    full[..., :k] = codes
    return _dev(full)[..., :k]


def _near(got, want, tol, dtype, label=""):
    """|got - want| within tol and the rounding of the type; infinities and NaN where the plain form has them."""
    with np.errstate(all="ignore"):
        top = {"bf16": 3.3895e38, "f16": 65504.0, "f32": 3.4028e38}[dtype]
        assert np.array_equal(np.isnan(got), np.isnan(want)), f"{label}: NaN pattern differs"
        fine = ~np.isnan(want) & (np.abs(want) + tol < top)
        err = np.abs(got - want) - tol - R.EPS[dtype] * (np.abs(want) + tol) - R.TINY[dtype]
    bad = fine & ~(err <= 0)
    assert not bad.any(), f"{label}: {bad.sum()} of {bad.size}, first {np.argwhere(bad)[0]}: {got[bad][0]!r} for {want[bad][0]!r} +- {np.broadcast_to(tol, want.shape)[bad][0]!r}"


# ---------------------------------------------------------------- quantize

def _quantize(F, x, dtype, gated=False, blocks_first=False, x_pad=0, row_count=None):
    """The kernel's codes and scales of x (values of the type), poisoned before."""
    rows, k = x.shape[0], x.shape[1] // (2 if gated else 1)
    t = torch.zeros(rows, x.shape[1] + x_pad, dtype=DT[dtype], device="cuda")
    t[:, :x.shape[1]] = _dev(x, DT[dtype])
    codes = torch.full((rows, -(-k // 16) * 16 + 16), 0xaa, dtype=torch.uint8, device="cuda")
    n = F.blocks(k)
    scales = torch.full((n, rows) if blocks_first else (rows, n), -7.0, device="cuda")
    scales = scales.t() if blocks_first else scales
    F.Fp8Quantize(t[:, :x.shape[1]], codes[:, :k], scales, gated=gated, row_count=None if row_count is None else _ints([row_count])).encode()
    torch.cuda.synchronize()
    assert (codes[:, k:] == 0xaa).all(), "bytes behind a row's end were written"
    return codes[:, :k].cpu().numpy(), scales.cpu().numpy()


def _held(x, dtype):
    return torch.from_numpy(x).to(DT[dtype]).double().numpy()


def _check_codes(got, want):
    (c, s), (cw, sw) = got, want
    assert np.array_equal(np.isnan(s), np.isnan(sw)) and np.array_equal(np.nan_to_num(s), np.nan_to_num(sw))
    bad = c != cw
    assert not bad.any(), f"{bad.sum()} of {bad.size} codes, first {np.argwhere(bad)[0]}: {c[bad][0]} for {cw[bad][0]}"


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,k,pad,first", [(1, 1, 0, False), (3, 127, 0, False), (5, 128, 8, True), (2, 129, 3, False), (17, 256, 0, True),
                                              (64, 1000, 0, False), (33, 4096, 0, False), (300, 72, 0, True), (1, 8200, 0, False)])
def test_quantize(F, dtype, rows, k, pad, first):
    r = np.random.default_rng(rows * 1000 + k)
    x = _held(r.normal(0, 1, (rows, k)) * np.exp(r.normal(0, 2, (rows, 1))), dtype)
    x[r.random(x.shape) < 0.01] *= 20
    x = _held(x, dtype)
    _check_codes(_quantize(F, x, dtype, blocks_first=first, x_pad=pad), R.quantize(x))


def test_quantize_many_values(F):
    """A million f32 values, and values at and beside the middles of two codes under scales that are no powers of two."""
    r = np.random.default_rng(1)
    x = r.normal(0, 1, (1024, 1024)).astype(np.float32).astype(np.float64)
    _check_codes(_quantize(F, x, "f32"), R.quantize(x))
    top = r.uniform(1, 2, (512, 1)).astype(np.float32)
    scale = (top.astype(np.float64) / 448).astype(np.float32)
    near = (R._MIDDLE[None, :] * scale.astype(np.float64)).astype(np.float32)
    x = np.concatenate([top, near, np.zeros((512, 1), np.float32)], 1)
    for step in (np.float32(0), np.float32(np.inf), np.float32(-np.inf)):
        y = (x if step == 0 else np.concatenate([top, np.nextafter(near, step), np.zeros((512, 1), np.float32)], 1)).astype(np.float64)
        y[::2] *= -1
        _check_codes(_quantize(F, y, "f32"), R.quantize(y))


def test_quantize_exact_ties(F):
    """A block whose largest is 448 has the scale 1: middles go to the even code."""
    x = np.concatenate([R._MIDDLE, [448.0, 0.0]])[None]
    got = _quantize(F, np.concatenate([x, -x]), "f32")
    _check_codes(got, R.quantize(np.concatenate([x, -x])))
    assert (got[0][0][:126] % 2 == 0).all()


def test_quantize_ends_of_the_range(F):
    x = np.zeros((12, 256))
    x[1, 3], x[1, 200] = 3e38, 1e-38
    x[2, :] = 2.0 ** -149
    x[3, :128] = np.arange(128) * 2.0 ** -140
    x[4, 5] = np.inf
    x[5, 130] = -np.inf
    x[6, 255] = np.nan
    x[7, 0], x[7, 1] = np.nan, np.inf
    x[8, :] = -0.0
    x[9, :128] = np.arange(128) * 2.0 ** -126 * 1.37
    x[10, :128] = np.linspace(0, 448 * 2.0 ** -126, 128)
    x[11, :] = -3.4e38
    x = x.astype(np.float32).astype(np.float64)
    got = _quantize(F, x, "f32")
    _check_codes(got, R.quantize(x))
    assert np.isnan(got[1][4]).tolist() == [True, False] and np.isnan(got[1][5]).tolist() == [False, True]


@pytest.mark.parametrize("count", [-5, 0, 1, 7, 20, 2 ** 31 - 1])
def test_quantize_leaves_rows_behind_the_count(F, count):
    x = _held(np.random.default_rng(2).normal(0, 1, (20, 300)), "bf16")
    codes, scales = _quantize(F, x, "bf16", row_count=count)
    n = min(max(count, 0), 20)
    want = R.quantize(x)
    _check_codes((codes[:n], scales[:n]), (want[0][:n], want[1][:n]))
    assert (codes[n:] == 0xaa).all() and (scales[n:] == -7.0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,k,pad", [(3, 128, 0), (40, 768, 0), (9, 200, 0), (5, 131, 1)])
def test_quantize_gated(F, dtype, rows, k, pad):
    """value * silu(gate) is computed in f32: some ten roundings of 2^-24 and an exponential of 2^-22, 2^-20 in all. So scales are
    off by 2^-20 of themselves at most, and a code's value by half a step of its binade and 2^-19 of the value."""
    r = np.random.default_rng(k)
    x = _held(r.normal(0, 2, (rows, 2 * k)) * np.exp(r.normal(0, 1, (rows, 1))), dtype)
    x[0, k:] = _held(np.linspace(-60, 60, k), dtype)
    codes, scales = _quantize(F, x, dtype, gated=True, x_pad=pad)
    y = R.gated(x)
    want = R.quantize(y)[1].astype(np.float64)
    assert (np.abs(scales - want) <= 2.0 ** -20 * want).all()
    s = R.spread(scales.astype(np.float64), k)
    v = R.VALUES[codes] * s
    step = np.maximum(2.0 ** np.floor(np.log2(np.maximum(np.abs(y) / s, 2.0 ** -6))), 2.0 ** -6) / 8
    assert (np.abs(v - y) <= s * step / 2 * (1 + 2.0 ** -18) + 2.0 ** -19 * np.abs(y)).all()


def test_quantize_gated_ends(F):
    """Gates far below zero give zeros, infinities and NaN spoil their block only."""
    x = np.zeros((5, 512))
    x[:, :256] = 1.0
    x[0, 256:] = -300.0
    x[1, 256:] = 300.0
    x[2, 256] = np.inf
    x[3, 500] = np.nan
    x[4, 10] = np.inf
    codes, scales = _quantize(F, x, "f32", gated=True)
    assert (R.VALUES[codes[0]] == 0).all() and scales[0].max() <= R.SMALLEST_SCALE
    assert (codes[1] == 126).all() and np.allclose(scales[1], 300 / 448, rtol=1e-6)
    assert np.isnan(scales[2]).tolist() == [True, False] and np.isnan(scales[3]).tolist() == [False, True]
    assert np.isnan(scales[4]).tolist() == [True, False] and (codes[2, :128] == 0).all()


# ---------------------------------------------------------------- products

def _operands(r, m, n, k, lead=()):
    def codes(*shape):
        c = R.nearest(r.normal(0, 110, shape))
        return np.where(r.random(shape) < 0.02, r.integers(0, 127, shape), c).astype(np.uint8)

    a, b = codes(m, k), codes(*lead, n, k)
    sa = (0.01 * np.exp(r.normal(0, 1, (m, R.blocks(k))))).astype(np.float32)
    sb = (2e-4 * np.exp(r.normal(0, 1, lead + (R.blocks(n), R.blocks(k))))).astype(np.float32)
    return a, sa, b, sb


def _epilogue(sum_, tol, ab, old, bias, cap):
    """The other operations on the sums and their bound: an f32 rounding each of what it works on."""
    v = ab * sum_
    tol = tol + 2.0 ** -24 * np.abs(v)
    for more in (old, bias):
        if more is not None:
            tol = tol + 2.0 ** -24 * (np.abs(v) + np.abs(more))
            v = v + more
    if cap is not None:
        v = cap * np.tanh(v / cap)
        tol = tol + 2.0 ** -21 * cap
    return v, tol


SIZES = [(1, 1, 1), (1, 16, 128), (1, 300, 1000), (2, 129, 256), (3, 64, 130), (5, 130, 200), (16, 128, 128), (17, 127, 384), (31, 257, 512),
         (33, 96, 2048), (64, 256, 144), (65, 200, 640), (100, 33, 4096), (128, 128, 1024), (129, 385, 272), (200, 1000, 257), (300, 520, 1536)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul(F, dtype, m, n, k):
    r = np.random.default_rng(m * 10007 + n * 101 + k)
    a, sa, b, sb = _operands(r, m, n, k)
    d = torch.full((m, n), 7.0, dtype=DT[dtype], device="cuda")
    F.Fp8Matmul(_padded(a), _dev(sa), _padded(b), _dev(sb), d).encode()
    torch.cuda.synchronize()
    want, mag, cut = R.product(a, sa, b, sb)
    _near(_np(d), want, R.bound(want, mag, cut, k, dtype), dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,n,k", [(1, 200, 256), (6, 130, 384), (70, 190, 300)])
@pytest.mark.parametrize("ab,accumulate,bias,cap", [(0.5, True, False, None), (-2.0, False, True, None), (1.0, True, True, 0.3),
                                                    (3.0, False, False, 30.0)])
def test_matmul_epilogue_and_strides(F, dtype, m, n, k, ab, accumulate, bias, cap):
    """D-ops, rows with gaps, scales with their blocks outermost, and a d whose rows start at odd places; what is between d's rows
    stays."""
    r = np.random.default_rng(m + n + k)
    a, sa, b, sb = _operands(r, m, n, k)
    wide = torch.zeros(m, -(-k // 16) * 16 + 48, dtype=torch.uint8, device="cuda") + 0x7f
    wide[:, :k] = _dev(a)
    old, bi = _held(r.normal(0, 1, (m, n)), dtype), _held(r.normal(0, 1, n), dtype)
    full = torch.full((m, n + 3), 5.0, dtype=DT[dtype], device="cuda")
    d = full[:, 1:n + 1]
    d.copy_(_dev(old, DT[dtype]))
    F.Fp8Matmul(wide[:, :k], _dev(sa.T).t(), _padded(b), _dev(sb.T).t(), d, bias=_dev(bi, DT[dtype]) if bias else None, ab_scale=ab,
                accumulate=accumulate, soft_cap=cap).encode()
    torch.cuda.synchronize()
    assert (full[:, 0] == 5).all() and (full[:, n + 1:] == 5).all()
    want, mag, cut = R.product(a, sa, b, sb)
    want, tol = _epilogue(want, R.bound(want, mag, cut, k, dtype, ab), ab, old if accumulate else None, bi if bias else None, cap)
    _near(_np(d), want, tol, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,n,k", [(64, 1024, 8192), (70, 1001, 6000), (17, 300, 16384), (130, 516, 8200)])
def test_matmul_in_parts(F, dtype, m, n, k):
    """Products whose inner axis is shared by workgroups, with a bias and another operator's call between two on one workspace."""
    r = np.random.default_rng(m + n)
    a, sa, b, sb = _operands(r, m, n, k)
    bias = _held(r.normal(0, 1, n), dtype)
    x = [_padded(a), _dev(sa), _padded(b), _dev(sb)]
    d, e = (torch.full((m, n), 7.0, dtype=DT[dtype], device="cuda") for _ in range(2))
    first = F.Fp8Matmul(*x, d, bias=_dev(bias, DT[dtype]))
    assert first.workspace_bytes > 0
    second = F.Fp8Matmul(*x, e, ab_scale=2.0, workspace=first.workspace)
    for op in (first, second, first):
        op.encode()
    torch.cuda.synchronize()
    want, mag, cut = R.product(a, sa, b, sb)
    for t, ab, bi in ((d, 1.0, bias), (e, 2.0, None)):
        w, tol = _epilogue(want, R.bound(want, mag, cut, k, dtype, ab), ab, None, bi, None)
        _near(_np(t), w, tol, dtype)


def test_captured_products_in_parts(F):
    """Two captured calls with workspaces of their own replay on other rows."""
    r = np.random.default_rng(14)
    m, n, k = 64, 512, 8192
    a, sa, b, sb = _operands(r, m, n, k)
    sets = []
    for _ in range(2):
        x = [_padded(a), _dev(sa), _padded(b), _dev(sb), torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")]
        op = F.Fp8Matmul(*x)
        assert op.workspace_bytes > 0
        op.encode()
        sets.append((x, op))
    torch.cuda.synchronize()
    graphs, stream = [], torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    for _, op in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            op.encode()
        graphs.append(g)
    for _ in range(3):
        wants = []
        for x, _ in sets:
            a = R.nearest(r.normal(0, 110, (m, k)))
            x[0].copy_(_dev(a))
            wants.append(R.product(a, sa, b, sb))
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (x, _), (want, mag, cut) in zip(sets, wants):
            _near(_np(x[4]), want, R.bound(want, mag, cut, k, "bf16"), "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", [(300, 3000, 1160), (1500, 4100, 136), (1501, 4103, 1160), (3000, 8200, 136), (3001, 8203, 136), (2500, 8200, 2304)])
def test_matmul_wide_tiles(F, dtype, m, n, k):
    """Calls of tiles of 64, 128 and 256, their last row and column tiles cut, odd strides among them; some rows are compared."""
    r = np.random.default_rng(m)
    a, sa, b, sb = _operands(r, m, n, k)
    d = torch.full((m, n), 7.0, dtype=DT[dtype], device="cuda")
    F.Fp8Matmul(_padded(a), _dev(sa), _padded(b), _dev(sb), d).encode()
    torch.cuda.synchronize()
    assert not (d == 7).all(1).any()
    at = np.unique(np.concatenate([np.arange(0, m, max(7, m // 60)), [m - 1]]))
    want, mag, cut = R.product(a[at], sa[at], b, sb)
    _near(_np(d)[at], want, R.bound(want, mag, cut, k, dtype), dtype)


@pytest.mark.parametrize("m,n,k", [(1, 130, 512), (5, 64, 256), (150, 200, 384)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_matmul_not_a_number(F, dtype, m, n, k):
    """NaN codes and scales reach their own row or column (or block of columns) and no other; infinite scales too."""
    r = np.random.default_rng(9)
    a, sa, b, sb = _operands(r, m, n, k)
    a[0, 200] = 0x7f
    b[3, 7] = 0xff
    sb[0, 1] = np.inf if m > 1 else sb[0, 1]
    sa[m - 1, 0] = np.nan if m > 1 else sa[0, 0]
    d = torch.zeros(m, n, dtype=DT[dtype], device="cuda")
    F.Fp8Matmul(_padded(a), _dev(sa), _padded(b), _dev(sb), d).encode()
    torch.cuda.synchronize()
    with np.errstate(all="ignore"):
        want, mag, cut = R.product(a, sa, b, sb)
        got = _np(d)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        fine = np.isfinite(want)
        assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
        tol = np.where(np.isfinite(mag + cut), R.bound(want, mag, cut, k, dtype), 0.0)
    _near(np.where(fine, got, 0.0), np.where(fine, want, 0.0), np.where(fine, tol, 0.0), dtype)


def test_matmul_large_scales(F):
    """Scales from the quantizer's smallest to large ones, products that leave f16, and sums in f32's range."""
    r = np.random.default_rng(10)
    a, sa, b, sb = _operands(r, 20, 140, 256)
    sa[0], sa[1], sa[2] = 2.0 ** -126, 1e30, 1e36
    sb *= 1e3
    for dtype in ("f16", "bf16", "f32"):
        d = torch.zeros(20, 140, dtype=DT[dtype], device="cuda")
        F.Fp8Matmul(_padded(a), _dev(sa), _padded(b), _dev(sb), d).encode()
        torch.cuda.synchronize()
        want, mag, cut = R.product(a, sa, b, sb)
        tol = R.bound(want, mag, cut, 256, dtype) + 2.0 ** -149 * 3 * 128 * 448 * 448
        # A partial sum is at most the sum of the magnitudes. Where that passes f32's largest value, 3.4e38, a partial sum may be
        # infinite though the whole is not: sums are f32, and such outputs (of the row of scale 1e36) are not compared.
        held = mag * (1 + 2.0 ** -15) < 3.4e38
        assert held[np.arange(20) != 2].all()
        _near(np.where(held, _np(d), 0.0), np.where(held, want, 0.0), np.where(held, tol, 0.0), dtype)


# ---------------------------------------------------------------- grouped products

def _grouped(F, r, sizes, n, k, dtype, gather, spare=0, lead_rows=0, bias=False, tokens=50, every=1):
    E, total = len(sizes), sum(sizes)
    m = lead_rows + total + spare
    start = lead_rows + np.concatenate([[0], np.cumsum(sizes)])
    count = tokens if gather else m
    a, sa, b, sb = _operands(r, count, n, k, (E,))
    rows = r.integers(0, tokens, m) if gather else None
    bi = _held(r.normal(0, 1, (E, n)), dtype) if bias else None
    d = torch.full((m, n), 3.0, dtype=DT[dtype], device="cuda")
    op = F.Fp8GroupedMatmul(_padded(a), _dev(sa), _padded(b), _dev(sb), d, _ints(start), a_rows=_ints(rows) if gather else None,
                            bias=_dev(bi, DT[dtype]) if bias else None)
    op.encode()
    torch.cuda.synchronize()
    got = _np(d)
    live = np.zeros(m, bool)
    for e in range(E):
        at = slice(start[e], start[e + 1])
        live[at] = True
        if sizes[e] == 0:
            continue
        some = np.unique(np.concatenate([np.arange(start[e], start[e + 1], every), [start[e + 1] - 1]]))
        which = rows[some] if gather else some
        want, mag, cut = R.product(a[which], sa[which], b[e], sb[e])
        want, tol = _epilogue(want, R.bound(want, mag, cut, k, dtype), 1.0, None, bi[e] if bias else None, None)
        _near(got[some], want, tol, dtype, f"expert {e}")
        assert not (got[at] == 3).all(1).any()
    assert (got[~live] == 3).all(), "rows of no group were written"


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("sizes,n,k", [([1], 64, 128), ([0, 0, 3], 130, 256), ([1, 0, 2, 1, 1, 0, 1], 256, 200), ([5, 16, 17, 0, 1], 100, 384),
                                       ([130, 1, 0, 260], 200, 272), ([40, 200, 7], 300, 512), ([0, 0], 64, 128)])
def test_grouped(F, dtype, gather, sizes, n, k):
    _grouped(F, np.random.default_rng(sum(sizes) + n), sizes, n, k, dtype, gather)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_grouped_wide_tiles(F, dtype):
    _grouped(F, np.random.default_rng(15), [900, 0, 1030, 513, 257, 1, 2300], 4100, 136, dtype, True, spare=9, tokens=300, every=23)


@pytest.mark.parametrize("gather", [False, True])
def test_grouped_rows_of_no_group(F, gather):
    _grouped(F, np.random.default_rng(11), [3, 0, 70, 9], 130, 260, "bf16", gather, spare=37, lead_rows=5, bias=True)


@pytest.mark.parametrize("experts,most", [(64, 3), (65, 2), (200, 40), (1024, 2)])
def test_grouped_many_experts(F, experts, most):
    r = np.random.default_rng(experts)
    _grouped(F, r, [int(x) for x in r.integers(0, most + 1, experts)], 40, 128, "bf16", True, spare=3)


def test_grouped_bad_starts_and_rows(F):
    """Starts before, behind and out of order are cut to the rows; a row of a that is not there gives NaN."""
    r = np.random.default_rng(12)
    a, sa, b, sb = _operands(r, 10, 64, 128, (4,))
    rows = np.array([0, 1, 2, -1, 10, 2 ** 31 - 1, 9, 3, 4, 5, 6, 7])
    d = torch.full((12, 64), 3.0, device="cuda")
    F.Fp8GroupedMatmul(_padded(a), _dev(sa), _padded(b), _dev(sb), d, _ints([-4, 8, 6, 6, 99]), a_rows=_ints(rows)).encode()
    torch.cuda.synchronize()
    got = _np(d)
    assert np.isnan(got[3:6]).all() and np.isfinite(np.delete(got, [3, 4, 5], 0)).all()
    for e, at in ((0, [0, 1, 2]), (3, [8, 9, 10, 11])):
        want, mag, cut = R.product(a[rows[at]], sa[rows[at]], b[e], sb[e])
        _near(got[at], want, R.bound(want, mag, cut, 128, "f32"), "f32")


def test_grouped_is_the_dense_product(F):
    """One group of all rows gives the dense call's bits where both take the same kernel, and its values anyway."""
    r = np.random.default_rng(13)
    a, sa, b, sb = _operands(r, 300, 200, 640, (1,))
    x = [_padded(a), _dev(sa), _padded(b), _dev(sb)]
    d, g = torch.zeros(300, 200, device="cuda"), torch.zeros(300, 200, device="cuda")
    F.Fp8Matmul(x[0], x[1], x[2][0], x[3][0], d).encode()
    F.Fp8GroupedMatmul(*x, g, _ints([0, 300])).encode()
    torch.cuda.synchronize()
    want, mag, cut = R.product(a, sa, b[0], sb[0])
    for t in (d, g):
        _near(_np(t), want, R.bound(want, mag, cut, 640, "f32"), "f32")


# ---------------------------------------------------------------- plan and combine

@pytest.mark.parametrize("tokens,active,routed,experts,first", [
    (0, 2, 8, 8, 0), (1, 1, 1, 1, 0), (1, 8, 128, 128, 0), (16, 8, 128, 128, 0), (7, 3, 5, 2, 3), (64, 1, 64, 64, 0), (65, 1, 63, 63, 0),
    (1000, 8, 128, 128, 0), (1024, 8, 512, 128, 384), (1025, 8, 1024, 1024, 0), (3000, 4, 60, 60, 0), (8192, 8, 128, 128, 0),
    (20000, 2, 300, 100, 100), (5000, 8, 1, 1, 0)])
def test_plan(F, tokens, active, routed, experts, first):
    ids = np.random.default_rng(tokens + experts).integers(0, routed, (tokens, active))
    if tokens > 3 and routed > 4:
        ids[::3] = ids[::3] % 3  # some experts are liked far more
    t = _ints(ids).view(tokens, active)
    op = F.ExpertPlan(t, experts, first)
    for _ in range(2):
        for x in (op.group_start, op.tokens, op.slots):
            x.fill_(-99)
        op.encode()
        torch.cuda.synchronize()
        start, toks, slots = R.plan(ids, experts, first)
        assert np.array_equal(_np(op.group_start), start)
        assert np.array_equal(_np(op.tokens), toks)
        assert np.array_equal(_np(op.slots), slots)


def test_plan_of_ids_that_are_no_experts(F):
    ids = np.array([[-1, 3], [2 ** 31 - 1, 2], [5, -2 ** 31], [3, 3]])
    op = F.ExpertPlan(_ints(ids), 3, 2)
    op.encode()
    torch.cuda.synchronize()
    start, toks, slots = R.plan(ids, 3, 2)
    assert np.array_equal(_np(op.group_start), start) and np.array_equal(_np(op.tokens), toks) and np.array_equal(_np(op.slots), slots)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("tokens,active,rows,width,pad", [(1, 1, 1, 1, 0), (3, 8, 20, 2048, 0), (16, 8, 128, 1000, 0), (5, 2, 9, 77, 0), (70, 4, 100, 4096, 8),
                                                          (2, 9, 5, 333, 3), (1, 64, 40, 256, 0), (4, 3, 0, 64, 0)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_combine(F, dtype, tokens, active, rows, width, pad, accumulate):
    r = np.random.default_rng(tokens * 100 + width)
    x, old = _held(r.normal(0, 1, (rows, width)), dtype), _held(r.normal(0, 1, (tokens, width)), dtype)
    slots = r.integers(-2, rows + 2, (tokens, active))
    w = r.random((tokens, active)).astype(np.float32)
    w[(slots < 0) | (slots >= rows)] = np.nan  # what is not counted is not looked at
    xt = torch.zeros(rows, width + pad, dtype=DT[dtype], device="cuda")
    xt[:, :width] = _dev(x, DT[dtype])
    out = torch.full((tokens, width + pad), 9.0, dtype=DT[dtype], device="cuda")
    out[:, :width] = _dev(old, DT[dtype])
    F.ExpertCombine(xt[:, :width], _ints(slots).view(tokens, active), _dev(w), out[:, :width], accumulate).encode()
    torch.cuda.synchronize()
    assert (out[:, width:] == 9).all()
    want, mag = R.combine(x, slots, w.astype(np.float64), old if accumulate else None)
    _near(_np(out[:, :width]), want, mag * (active + 1) * 2.0 ** -24, dtype)


# ---------------------------------------------------------------- together

def _layer(F, r, tokens, model, hidden, experts, active, dtype="bf16", first=0, routed=None):
    """A routed layer's operators on one set of buffers, in order."""
    routes = tokens * active
    a, sa, up, up_s = _operands(r, 1, 2 * hidden, model, (experts,))
    _, _, down, down_s = _operands(r, 1, model, hidden, (experts,))
    s = dict(x=_dev(r.normal(0, 1, (tokens, model)), DT[dtype]), ids=_ints(r.integers(0, routed or experts, (tokens, active))),
             weights=_dev(r.random((tokens, active)).astype(np.float32)), out=torch.zeros(tokens, model, dtype=DT[dtype], device="cuda"),
             h=torch.zeros(routes, 2 * hidden, dtype=DT[dtype], device="cuda"), y=torch.zeros(routes, model, dtype=DT[dtype], device="cuda"))
    s["codes"], s["scales"] = F.new_rows(tokens, model)
    s["h_codes"], s["h_scales"] = F.new_rows(routes, hidden)
    plan = F.ExpertPlan(s["ids"], experts, first)
    s["plan"] = plan
    up_s, down_s = up_s * 20, down_s * 20
    s["w"] = (up, up_s, down, down_s)
    s["ops"] = [plan, F.Fp8Quantize(s["x"], s["codes"], s["scales"]),
                F.Fp8GroupedMatmul(s["codes"], s["scales"], _padded(up), _dev(up_s), s["h"], plan.group_start, a_rows=plan.tokens),
                F.Fp8Quantize(s["h"], s["h_codes"], s["h_scales"], gated=True, row_count=plan.count),
                F.Fp8GroupedMatmul(s["h_codes"], s["h_scales"], _padded(down), _dev(down_s), s["y"], plan.group_start),
                F.ExpertCombine(s["y"], plan.slots, s["weights"], s["out"])]
    return s


def _layer_check(s, tokens, active, experts, first=0):
    """Each operator against its plain form on what the one before it gave."""
    up, up_s, down, down_s = s["w"]
    ids = _np(s["ids"])
    start, toks, slots = R.plan(ids, experts, first)
    assert np.array_equal(_np(s["plan"].group_start), start) and np.array_equal(_np(s["plan"].slots), slots)
    live = start[-1]
    codes, scales = R.quantize(_np(s["x"]))
    got = s["codes"].view(torch.uint8).cpu().numpy()
    _check_codes((got, s["scales"].cpu().numpy()), (codes, scales))
    h, y = _np(s["h"]), _np(s["y"])
    hc, hs = s["h_codes"].view(torch.uint8).cpu().numpy(), s["h_scales"].cpu().numpy()
    for e in range(experts):
        at = slice(start[e], start[e + 1])
        if start[e] == start[e + 1]:
            continue
        want, mag, cut = R.product(codes[toks[at]], scales[toks[at]], up[e], up_s[e])
        _near(h[at], want, R.bound(want, mag, cut, up.shape[2], "bf16"), "bf16", f"up {e}")
        want, mag, cut = R.product(hc[at], hs[at], down[e], down_s[e])
        _near(y[at], want, R.bound(want, mag, cut, down.shape[2], "bf16"), "bf16", f"down {e}")
    g = R.gated(h[:live])
    k = g.shape[1]
    v = R.VALUES[hc[:live]] * R.spread(hs[:live].astype(np.float64), k)
    s_ = R.spread(hs[:live].astype(np.float64), k)
    step = np.maximum(2.0 ** np.floor(np.log2(np.maximum(np.abs(g) / s_, 2.0 ** -6))), 2.0 ** -6) / 8
    assert (np.abs(v - g) <= s_ * step / 2 * (1 + 2.0 ** -18) + 2.0 ** -19 * np.abs(g)).all()
    want, mag = R.combine(y, slots, _np(s["weights"]))
    _near(_np(s["out"]), want, mag * (active + 1) * 2.0 ** -24, "bf16")


@pytest.mark.parametrize("tokens,model,hidden,experts,active,first,routed", [(1, 256, 128, 8, 2, 0, 8), (40, 384, 200, 6, 3, 0, 6),
                                                                             (300, 256, 144, 4, 2, 0, 4), (50, 256, 128, 4, 4, 4, 16)])
def test_a_routed_layer(F, tokens, model, hidden, experts, active, first, routed):
    s = _layer(F, np.random.default_rng(tokens), tokens, model, hidden, experts, active, first=first, routed=routed)
    for op in s["ops"]:
        op.encode()
    torch.cuda.synchronize()
    _layer_check(s, tokens, active, experts, first)


def test_a_captured_layer(F):
    """Two layers captured on a stream of their own replay with other routes and rows, with eager work between the replays."""
    r = np.random.default_rng(20)
    tokens, experts, active = 24, 5, 3
    layers = [_layer(F, r, tokens, 256, 128, experts, active) for _ in range(2)]
    for s in layers:
        for op in s["ops"]:
            op.encode()
    torch.cuda.synchronize()
    graphs, stream = [], torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    for s in layers:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            for op in s["ops"]:
                op.encode()
        graphs.append(g)
    for i in range(4):
        for s in layers:
            s["x"].copy_(_dev(r.normal(0, 1, tuple(s["x"].shape)), torch.bfloat16))
            s["ids"].copy_(_ints(r.integers(0, experts + (i == 3), (tokens, active))))
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for s in layers:
            _layer_check(s, tokens, active, experts)
        eager = _layer(F, r, 3, 256, 128, experts, active)
        for op in eager["ops"]:
            op.encode()
        torch.cuda.synchronize()
        _layer_check(eager, 3, active, experts)


def test_calls_on_two_streams(F):
    """Operators on streams other than the tensors' own, at once, each with buffers of its own; a call repeated gives its bits."""
    r = np.random.default_rng(21)
    streams = [torch.cuda.Stream() for _ in range(2)]
    layers = [_layer(F, r, 60, 256, 128, 7, 2) for _ in streams]
    torch.cuda.synchronize()
    first = []
    for _ in range(3):
        for st, s in zip(streams, layers):
            for op in s["ops"]:
                op.encode(stream=st)
    torch.cuda.synchronize()
    for s in layers:
        _layer_check(s, 60, 2, 7)
        first.append(s["out"].clone())
    for st, s, was in zip(streams, layers, first):
        with torch.cuda.stream(st):
            for op in s["ops"]:
                op.encode()
        st.synchronize()
        assert torch.equal(s["out"], was)


def test_calls_of_nothing(F):
    """No rows, no columns, no tokens: nothing is launched or written, and a plan's starts are zeros."""
    w, ws = F.new_rows(8, 200)
    ws = torch.zeros(1, 2, device="cuda")
    c0, s0 = F.new_rows(0, 200)
    F.Fp8Matmul(c0, s0, w, ws, torch.zeros(0, 8, device="cuda")).encode()
    c, s = F.new_rows(5, 200)
    F.Fp8Matmul(c, s, w[:0], torch.zeros(0, 2, device="cuda"), torch.zeros(5, 0, device="cuda")).encode()
    F.Fp8GroupedMatmul(c0, s0, w[None], ws[None], torch.zeros(0, 8, device="cuda"), _ints([0, 0])).encode()
    F.Fp8Quantize(torch.zeros(0, 200, device="cuda"), c0, s0).encode()
    plan = F.ExpertPlan(torch.zeros(0, 2, dtype=torch.int32, device="cuda"), 3)
    plan.group_start.fill_(-1)
    plan.encode()
    F.ExpertCombine(torch.zeros(0, 8, device="cuda"), torch.zeros(0, 2, dtype=torch.int32, device="cuda"), torch.zeros(0, 2, device="cuda"),
                    torch.zeros(0, 8, device="cuda")).encode()
    torch.cuda.synchronize()
    assert plan.group_start.tolist() == [0, 0, 0, 0]


def _far(F, shape):
    """Codes of more than 4 GiB, and their values' rows as float64 on the device."""
    c = torch.randint(0, 0x7f, shape, dtype=torch.uint8, device="cuda")
    c[:, ::2] |= 0x80
    return c, lambda rows: torch.from_numpy(R.VALUES).cuda()[c[rows].long()]


@pytest.mark.parametrize("m", [3, 40])
def test_matmul_places_past_32_bits(F, m):
    """Weights of 5.4 GB: the first and the last columns, in each kernel."""
    n, k = 41000, 131072
    c, values = _far(F, (n, k))
    a, sa = R.nearest(np.random.default_rng(1).normal(0, 110, (m, k))), np.full((m, k // 128), 1e-3, np.float32)
    d = torch.zeros(m, n, device="cuda")
    F.Fp8Matmul(_padded(a), _dev(sa), c, torch.full((R.blocks(n), k // 128), 1e-3, device="cuda"), d).encode()
    torch.cuda.synchronize()
    at = torch.tensor([0, 1, 20000, n - 33, n - 1], device="cuda")
    x = torch.from_numpy(R.VALUES[a]).cuda()
    scale = float(np.float32(1e-3)) ** 2
    want, mag = x @ values(at).t() * scale, x.abs() @ values(at).abs().t() * scale
    tol = R.bound(None, mag, 0, k, "f32")
    assert ((d[:, at].double() - want).abs() <= tol + 2.0 ** -24 * want.abs()).all()


def test_rows_past_32_bits(F):
    """Rows of more than 4 GiB in and out of the quantizer, the products and the sums: the last ones."""
    rows, k = 1100000, 4096
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    r = np.random.default_rng(2)
    last = _held(r.normal(0, 1, (40, k)), "bf16")
    x[-40:] = _dev(last, torch.bfloat16)
    codes, scales = F.new_rows(rows, k)
    F.Fp8Quantize(x, codes, scales).encode()
    torch.cuda.synchronize()
    want = R.quantize(last)
    _check_codes((codes[-40:].view(torch.uint8).cpu().numpy(), scales[-40:].cpu().numpy()), want)
    _, _, b, sb = _operands(r, 1, 4100, k)
    d = torch.zeros(rows, 4100, dtype=torch.bfloat16, device="cuda")
    F.Fp8Matmul(codes, scales, _padded(b), _dev(sb), d).encode()
    torch.cuda.synchronize()
    w, mag, cut = R.product(*want, b, sb)
    _near(_np(d[-40:]), w, R.bound(w, mag, cut, k, "bf16"), "bf16")
    out = torch.zeros(3, k, dtype=torch.bfloat16, device="cuda")
    slots = np.array([[rows - 1, 0], [rows - 40, rows - 2], [5, rows]])
    F.ExpertCombine(x, _ints(slots), _dev(np.ones((3, 2), np.float32)), out).encode()
    torch.cuda.synchronize()
    z = np.concatenate([last, np.zeros((1, k))])
    s, m = R.combine(z, np.array([[39, 40], [0, 38], [40, 41]]), np.ones((3, 2)))
    _near(_np(out), s, m * 3 * 2.0 ** -24, "bf16")


def test_python_refusals(F, qmm):
    codes, scales = F.new_rows(4, 200)
    w, ws = F.new_rows(6, 200)
    ws = torch.zeros(1, 2, device="cuda")
    d = torch.zeros(4, 6, device="cuda")

    def refused(fn, status=qmm.INVALID_ARGUMENT):
        with pytest.raises(qmm.MatmulError) as e:
            fn()
        assert e.value.status == status

    F.Fp8Matmul(codes, scales, w, ws, d)
    refused(lambda: F.Fp8Matmul(codes, scales[:, :1], w, ws, d))
    refused(lambda: F.Fp8Matmul(codes, scales, w, ws.double(), d))
    refused(lambda: F.Fp8Matmul(codes.float(), scales, w, ws, d))
    refused(lambda: F.Fp8Matmul(codes, scales, w[:, :199], ws, d))
    refused(lambda: F.Fp8Matmul(codes, scales, w, ws, d.double()), qmm.UNSUPPORTED_DATA_TYPE)
    refused(lambda: F.Fp8Matmul(codes, scales, w, ws, d.t()))
    refused(lambda: F.Fp8Matmul(codes, scales, w, ws, d, bias=torch.zeros(6, device="cuda", dtype=torch.bfloat16)))
    # rows that are not on 16-byte boundaries, and memory that ends before one
    tight = torch.zeros(4, 200, dtype=torch.uint8, device="cuda")
    refused(lambda: F.Fp8Matmul(tight, scales, w, ws, d))
    short = torch.zeros(3 * 208 + 200, dtype=torch.uint8, device="cuda").as_strided((4, 200), (208, 1))
    refused(lambda: F.Fp8Matmul(short, scales, w, ws, d))
    refused(lambda: F.Fp8Quantize(torch.zeros(4, 200, device="cuda"), codes, scales, gated=True))
    refused(lambda: F.ExpertPlan(torch.zeros(4, 2, dtype=torch.int64, device="cuda"), 4))
    refused(lambda: F.ExpertPlan(torch.zeros(4, 2, dtype=torch.int32, device="cuda"), 0))
    refused(lambda: F.ExpertCombine(d, torch.zeros(4, 1, dtype=torch.int32, device="cuda"), torch.zeros(4, 1, device="cuda"),
                                    torch.zeros(4, 6, device="cuda", dtype=torch.float16)))
    with pytest.raises(ValueError):
        F.Fp8Matmul(codes.cpu(), scales, w, ws, d)
