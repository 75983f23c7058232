"""Products of 8-bit floating-point codes on the GPU in every kernel that takes them (tests/fp8_forms.py), against the plain 64-bit
forms of tests/fp8_ref.py."""
import numpy as np
import pytest
import torch

from tests import fp8_forms as K
from tests import fp8_ref as R
from tests.test_gpu_fp8 import (DT, F, _dev, _epilogue, _held, _ints, _layer, _layer_check, _near, _np, _operands,  # noqa: F401
                                _padded)  # (F is a fixture)

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


_POOL = R.nearest(np.random.default_rng(0).normal(0, 110, 1 << 16))


def _many(r, m, n, k, lead=()):
    """_operands of many values: codes drawn from a pool of normally distributed ones."""
    a, b = _POOL[r.integers(0, _POOL.size, (m, k))], _POOL[r.integers(0, _POOL.size, lead + (n, k))]
    sa = (0.01 * np.exp(r.normal(0, 1, (m, R.blocks(k))))).astype(np.float32)
    sb = (2e-4 * np.exp(r.normal(0, 1, lead + (R.blocks(n), R.blocks(k))))).astype(np.float32)
    return a, sa, b, sb


# ab_scale, accumulate, bias, soft cap, elements before d's first and between its rows
EPILOGUES = [(1.0, False, False, None, 0, 8), (0.5, True, False, None, 8, 8), (-2.0, False, True, None, 1, 3), (1.0, True, True, 0.3, 0, 8),
             (3.0, False, False, 30.0, 1, 2), (0.5, True, True, 3.0, 3, 3)]


def _d(r, m, n, dtype, before, gap):
    """d inside a poisoned tensor, its values, and a check that what is around it stays."""
    full = torch.full((m, before + n + gap), 5.0, dtype=DT[dtype], device="cuda")
    d = full[:, before:before + n]
    g = torch.Generator(device="cuda")
    g.manual_seed(int(r.integers(1 << 30)))
    d.copy_(torch.randn(m, n, generator=g, device="cuda"))

    def around():
        assert (full[:, :before] == 5).all() and (full[:, before + n:] == 5).all()
    return d, d.clone(), around


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("ab,accumulate,bias,cap,before,gap", EPILOGUES)
@pytest.mark.parametrize("size,want", K.CUT_TILES + K.ROWS + K.PARTS)
def test_epilogues(F, dtype, size, want, ab, accumulate, bias, cap, before, gap):
    """The d_ops in every kernel, into rows that can and that cannot be stored in pieces; scales with their blocks outermost."""
    m, n, k = size
    r = np.random.default_rng(m * 7 + n)
    a, sa, b, sb = _many(r, m, n, k)
    d, old, around = _d(r, m, n, dtype, before, gap)
    bi = _held(r.normal(0, 1, n), dtype)
    F.Fp8Matmul(_padded(a), _dev(sa.T).t(), _padded(b), _dev(sb.T).t(), d, bias=_dev(bi, DT[dtype]) if bias else None, ab_scale=ab,
                accumulate=accumulate, soft_cap=cap).encode()
    torch.cuda.synchronize()
    around()
    at = _some(m, 24)
    want, mag, cut = R.product(a[at], sa[at], b, sb)
    want, tol = _epilogue(want, R.bound(want, mag, cut, k, dtype, ab), ab, _np(old[at]) if accumulate else None, bi if bias else None, cap)
    _near(_np(d[at]), want, tol, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("size,want", K.CUT_TILES)
def test_not_a_number_in_tiles(F, dtype, size, want):
    """NaN codes and scales reach their row, column or block of columns and no other; an infinite scale too."""
    m, n, k = size
    r = np.random.default_rng(n)
    a, sa, b, sb = _many(r, m, n, k)
    a[70, 100], b[3, 7], sb[1, 1], sa[m - 1, 0] = 0x7f, 0xff, np.inf, np.nan
    d = torch.zeros(m, n, dtype=DT[dtype], device="cuda")
    F.Fp8Matmul(_padded(a), _dev(sa), _padded(b), _dev(sb), d).encode()
    torch.cuda.synchronize()
    assert torch.isnan(d).all(1).nonzero().flatten().tolist() == [70, m - 1] and torch.isnan(d).all(0).nonzero().flatten().tolist() == [3]
    at = np.unique(np.concatenate([_some(m, 20), [69, 70, 71]]))
    with np.errstate(all="ignore"):
        want, mag, cut = R.product(a[at], sa[at], b, sb)
        got, fine = _np(d)[at], np.isfinite(want)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
        tol = np.where(np.isfinite(mag + cut), R.bound(want, mag, cut, k, dtype), 0.0)
    _near(np.where(fine, got, 0.0), np.where(fine, want, 0.0), np.where(fine, tol, 0.0), dtype)


def _check_groups(d, old, start, rows, a, sa, b, sb, dtype, ab=1.0, accumulate=False, bias=None, cap=None):
    """The first and last rows of each group and some between, and every row that no group has."""
    tokens, free = len(a), torch.ones(len(d), dtype=torch.bool)
    for e in range(len(b)):
        lo, hi = start[e], start[e + 1]
        free[lo:hi] = False
        if lo == hi:
            continue
        at = np.unique(np.clip([lo, lo + 17, (lo + hi) // 2, hi - 2, hi - 1], lo, hi - 1))
        src = at if rows is None else rows[at]
        there = (src >= 0) & (src < tokens)
        src = np.where(there, src, 0)
        want, mag, cut = R.product(a[src], sa[src], b[e], sb[e])
        want, tol = _epilogue(np.where(there[:, None], want, np.nan), R.bound(want, mag, cut, a.shape[1], dtype, ab), ab,
                              _np(old[at]) if accumulate else None, None if bias is None else bias[e], cap)
        _near(_np(d[at]), want, np.where(there[:, None], tol, 0.0), dtype, f"expert {e}")
    assert torch.equal(d[free.cuda()], old[free.cuda()])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("gather,missing,epilogue", [(True, False, 0), (False, False, 0), (True, True, 0), (False, False, 2), (True, True, 3), (True, False, 5)])
@pytest.mark.parametrize("sizes,n,k,want", K.GROUPED)
def test_grouped(F, dtype, sizes, n, k, want, gather, missing, epilogue):
    """Ragged groups in every kernel: gathered rows and rows in place, rows of a that are not there, a bias of each expert, the other
    d_ops, and rows of d before the first and behind the last group."""
    ab, accumulate, bias, cap, before, gap = EPILOGUES[epilogue]
    r = np.random.default_rng(sum(sizes) + epilogue)
    E, total, lead = len(sizes), sum(sizes), 5
    m = total + K.AROUND
    start = lead + np.concatenate([[0], np.cumsum(sizes)])
    tokens = 333 if gather else m
    a, sa, b, sb = _many(r, tokens, n, k, (E,))
    rows = r.integers(0, tokens, m) if gather else None
    if missing:
        rows[r.random(m) < 0.2] = r.choice([-1, tokens, 2 ** 31 - 1])
        rows[start[1] - 1] = -1
    d, old, around = _d(r, m, n, dtype, before, gap)
    bi = _held(r.normal(0, 1, (E, n)), dtype) if bias else None
    F.Fp8GroupedMatmul(_padded(a), _dev(sa), _padded(b), _dev(sb), d, _ints(start), a_rows=_ints(rows) if gather else None,
                       bias=_dev(bi, DT[dtype]) if bias else None, ab_scale=ab, accumulate=accumulate, soft_cap=cap).encode()
    torch.cuda.synchronize()
    around()
    _check_groups(d, old, start, rows, a, sa, b, sb, dtype, ab, accumulate, bi, cap)


@pytest.mark.parametrize("tokens,active,routed,experts,n,k,want", K.SHARES)
def test_a_share_of_the_experts(F, tokens, active, routed, experts, n, k, want):
    """A rank's experts: the plan's rows are a part of those that there may be, the others stay."""
    r = np.random.default_rng(tokens)
    first = routed - experts
    ids = np.argsort(r.random((tokens, routed)), 1)[:, :active]
    plan = F.ExpertPlan(_ints(ids).view(tokens, active), experts, first)
    a, sa, b, sb = _many(r, tokens, n, k, (experts,))
    d, old, _ = _d(r, tokens * active, n, "bf16", 0, 0)
    plan.encode()
    F.Fp8GroupedMatmul(_padded(a), _dev(sa), _padded(b), _dev(sb), d, plan.group_start, a_rows=plan.tokens).encode()
    torch.cuda.synchronize()
    start, toks, _ = R.plan(ids, experts, first)
    assert 0 < start[-1] < tokens * active // 2
    _check_groups(d, old, start, toks, a, sa, b, sb, "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("size,want", K.CUT_TILES)
def test_one_group_gives_the_dense_bits(F, dtype, size, want):
    m, n, k = size
    a, sa, b, sb = _many(np.random.default_rng(4), m, n, k)
    x = [_padded(a), _dev(sa), _padded(b), _dev(sb)]
    d, g = (torch.full((m, n), 7.0, dtype=DT[dtype], device="cuda") for _ in range(2))
    F.Fp8Matmul(*x, d).encode()
    F.Fp8GroupedMatmul(x[0], x[1], x[2][None], x[3][None], g, _ints([0, m])).encode()
    torch.cuda.synchronize()
    assert torch.equal(d, g) and not (d == 7).all(1).any()


@pytest.mark.parametrize("tokens,experts,active", [(1, 8, 2), (37, 60, 4), (300, 16, 2)])
def test_routes_to_a_layer(F, qmm, tokens, experts, active):
    """The router's ids and weights, which are flat, go through the layer as views."""
    r = np.random.default_rng(tokens)
    ids, weights = qmm.moe_route(_dev(r.normal(0, 2, (tokens, experts)).astype(np.float32)), tokens, experts, active)
    s = _layer(F, r, tokens, 256, 144, experts, active)
    plan = F.ExpertPlan(ids.view(tokens, active), experts)
    quantize = s["ops"][1]
    up = F.Fp8GroupedMatmul(s["codes"], s["scales"], *(_padded(s["w"][0]), _dev(s["w"][1])), s["h"], plan.group_start, a_rows=plan.tokens)
    gate = F.Fp8Quantize(s["h"], s["h_codes"], s["h_scales"], gated=True, row_count=plan.count)
    down = F.Fp8GroupedMatmul(s["h_codes"], s["h_scales"], *(_padded(s["w"][2]), _dev(s["w"][3])), s["y"], plan.group_start)
    s["plan"], s["ids"], s["weights"] = plan, ids.view(tokens, active), weights.view(tokens, active)
    for op in (plan, quantize, up, gate, down, F.ExpertCombine(s["y"], plan.slots, s["weights"], s["out"])):
        op.encode()
    torch.cuda.synchronize()
    _layer_check(s, tokens, active, experts)
