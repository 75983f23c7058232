"""Plain arithmetic of the 8-bit floating-point products (csrc/fp8_layout.h, compiled for the CPU), their plain forms, and what
the entry points refuse before they touch a GPU."""
import ctypes as C
import functools
import os
import random
import subprocess
import tempfile

import numpy as np
import pytest

from tests import fp8_ref as R

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stark_amd", "csrc")
FAKE = 1 << 20

_WRAP = """
#include "fp8_layout.h"
extern "C" {
void group(int32_t a, int32_t b, uint32_t n, uint32_t* r) { const fp8::Range x = fp8::group(a, b, n); r[0] = x.first; r[1] = x.count; }
uint32_t row_tiles(uint32_t rows, uint32_t groups, uint32_t tile) { return fp8::row_tiles(rows, groups, tile); }
uint32_t tile_of(uint32_t i, uint32_t tiles) { return fp8::tile_of(i, tiles); }
void row_share(uint64_t t, uint32_t n, uint32_t k, uint32_t* r) { const fp8::RowShare x = fp8::row_share(t, n, k); r[0] = x.strips; r[1] = x.waves; }
void place(uint32_t i, uint32_t rows, uint32_t columns, uint32_t* r) { const fp8::Place x = fp8::place(i, rows, columns); r[0] = x.row; r[1] = x.column; }
void choose(uint32_t m, uint32_t n, uint32_t k, uint32_t g, int grouped, int exact, uint32_t* r) {
    const fp8::Choice c = fp8::choose(m, n, k, g, grouped, exact); r[0] = c.tile; r[1] = c.rows; r[2] = c.parts;
}
void split(uint32_t i, uint32_t b, uint32_t* r) { const fp8::Split x = fp8::split(i, b, fp8::inverse(b)); r[0] = x.row; r[1] = x.block; }
}
"""


@functools.lru_cache(None)
def rules():
    with tempfile.TemporaryDirectory() as d:
        src, lib = os.path.join(d, "fp8.cpp"), os.path.join(d, "fp8.so")
        with open(src, "w") as f:
            f.write(_WRAP)
        subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", CSRC, src, "-o", lib], check=True)
        return C.CDLL(lib)


def _pair(fn, *args):
    r = (C.c_uint32 * 2)()
    fn(*args, r)
    return tuple(r)


def test_groups_stay_inside_the_rows():
    L = rules()
    for a, b, n, want in ((0, 5, 10, (0, 5)), (-3, 5, 10, (0, 5)), (4, 4, 10, (4, 0)), (7, 5, 10, (7, 0)), (5, 99, 10, (5, 5)),
                          (99, 100, 10, (10, 0)), (-5, -1, 10, (0, 0)), (0, 2 ** 31 - 1, 2 ** 24, (0, 2 ** 24))):
        assert _pair(L.group, a, b, n) == want


def test_row_tiles_are_enough():
    L, r = rules(), random.Random(3)
    for _ in range(400):
        groups, tile = r.choice([1, 2, 3, 60, 128, 1024]), r.choice([16, 64, 128, 256])
        sizes = [r.choice([0, 1, r.randint(0, 3 * tile)]) for _ in range(groups)]
        rows = sum(sizes) + r.choice([0, 5])
        assert sum(-(-s // tile) for s in sizes) <= L.row_tiles(rows, groups, tile)


def test_every_tile_has_one_workgroup():
    L = rules()
    for tiles in (0, 1, 7, 8, 9, 63, 64, 65, 1000):
        got = [L.tile_of(i, tiles) for i in range((tiles + 7) // 8 * 8)]
        assert sorted(t for t in got if t < tiles) == list(range(tiles))


def test_every_tile_has_one_place():
    """Workgroups past the last tile have none: neither a row tile nor a column tile of theirs is there."""
    L = rules()
    for rows, columns in ((0, 3), (1, 1), (1, 5), (2, 9), (7, 1), (8, 3), (9, 4), (16, 48), (61, 7)):
        tiles = rows * columns
        seen = []
        for i in range((tiles + 7) // 8 * 8 + 8):
            row, column = _pair(L.place, L.tile_of(i, tiles), rows, columns)
            if row < rows:
                assert column < columns
                seen.append((row, column))
            else:
                assert row == rows
        assert sorted(seen) == [(r, c) for r in range(rows) for c in range(columns)]


def test_items_split_into_rows_and_blocks():
    L, r = rules(), random.Random(4)
    for blocks in (1, 2, 3, 6, 7, 31, 32, 96, 8191, 8192):
        for item in [0, 1, blocks - 1, blocks, 2 ** 32 - 1, 2 ** 32 - blocks] + [r.randrange(2 ** 32) for _ in range(200)]:
            assert _pair(L.split, item, blocks) == divmod(item, blocks)


def test_row_shares_fill_the_gpu_and_no_more():
    L = rules()
    L.row_share.argtypes = [C.c_uint64, C.c_uint32, C.c_uint32, C.c_void_p]
    assert _pair(L.row_share, 1, 12288, 4096) == (1, 4) and _pair(L.row_share, 1, 4096, 12288) == (1, 8)
    assert _pair(L.row_share, 128, 1536, 2048) == (2, 4) and _pair(L.row_share, 1, 16, 65536) == (1, 16)
    assert _pair(L.row_share, 1, 4096, 4096) == (1, 4) and _pair(L.row_share, 1, 16, 100) == (1, 2) and _pair(L.row_share, 2 ** 20, 2 ** 24, 128) == (2, 4)


def _choose(m, n, k, groups=1, grouped=False, exact=False):
    r = (C.c_uint32 * 3)()
    rules().choose(m, n, k, groups, int(grouped), int(exact), r)
    return tuple(r)


def test_each_kernel_takes_its_calls():
    """(tile, rows of the few-rows kernel, parts of the inner axis)."""
    assert _choose(1, 12288, 4096) == (0, 16, 1) and _choose(5, 4096, 12288) == (0, 16, 1) and _choose(4096, 12288, 4096) == (256, 0, 1)
    assert _choose(32, 12288, 4096)[0] == 64 and _choose(64, 4096, 12288) == (64, 0, 4) and _choose(16, 256, 16384)[2] == 8 and _choose(512, 4096, 4096) == (64, 0, 1)
    assert _choose(128, 1001, 2000) == (0, 32, 1) and _choose(1024, 4096, 4096) == (128, 0, 1)
    for tokens, want in ((16, 0), (64, 0), (256, 64), (2048, 128), (8192, 256)):
        assert _choose(8 * tokens, 1536, 2048, 128, True)[0] == want


def test_choices_are_what_the_kernels_take():
    """Blocks of fewer than 128 codes go to the few-rows kernel; parts are of calls without groups and have four steps each."""
    r = random.Random(8)
    for _ in range(3000):
        m, n, k = (int(2 ** r.uniform(0, e)) for e in (24, 24, 20))
        grouped = r.random() < 0.5
        groups = int(2 ** r.uniform(0, 10)) if grouped else 1
        exact = r.random() < 0.5
        tile, rows, parts = _choose(m, n, k, groups, grouped, exact)
        assert (tile, rows) in ((0, 16), (0, 32), (64, 0), (128, 0), (256, 0)) and not (exact and tile == 256)
        assert parts == 1 or (not grouped and tile and 4 * parts <= -(-k // 128))
        if k < 128:
            assert tile == 0


def test_plain_codes_are_the_nearest():
    r = np.random.default_rng(5)
    q = np.concatenate([r.normal(0, 100, 3000), r.normal(0, 0.01, 3000), [0.0, 448.0, 460.0, 1e9, 2.0 ** -10, 3 * 2.0 ** -10]])
    c = R.nearest(q)
    best = np.abs(R._POSITIVE[None, :] - np.minimum(np.abs(q), 448)[:, None]).min(1)
    assert np.array_equal(np.abs(R.VALUES[c] - np.clip(q, -448, 448)), best)
    assert R.nearest(np.array([2.0 ** -10]))[0] == 0 and R.nearest(np.array([3 * 2.0 ** -10]))[0] == 2  # ties to even
    assert np.array_equal(R.nearest(R._POSITIVE), np.arange(127))


def test_plain_plan_is_a_stable_sort():
    r = np.random.default_rng(6)
    for experts, first in ((5, 0), (3, 1), (100, 0), (70, 20)):
        ids = r.integers(0, 100, (40, 3))
        start, tokens, slots = R.plan(ids, experts, first)
        for e in range(experts):
            mine = tokens[start[e]:start[e + 1]]
            assert np.array_equal(mine, np.sort(mine)) and (ids[mine] == e + first).any(1).all()
        assert (tokens[start[-1]:] == -1).all()
        flat = slots.reshape(-1)
        assert np.array_equal(np.sort(flat[flat >= 0]), np.arange(start[-1]))


# ---------------------------------------------------------------- refusals

def _struct(cls, base, over):
    s = cls()
    s.struct_size = C.sizeof(s)
    for n, v in dict(base, **over).items():
        o, parts = s, n.split("__")
        for p in parts[:-1]:
            o = getattr(o, p)
        setattr(o, parts[-1], v)
    return s


QUANTIZE = dict(data_type=30, x=FAKE, x_row_stride=512, codes=FAKE + 2 ** 16, code_row_stride=512, scales=FAKE + 2 ** 17,
                scale_row_stride=4, scale_block_stride=1, rows=8, columns=512)


def test_quantize_refusals():
    from stark_amd import fp8 as F, qmm as Q
    call = Q.lib().stark_qmm_fp8_quantize

    def go(**kw):
        return call(C.byref(_struct(F._QuantizeArgs, QUANTIZE, kw)), None)

    assert call(None, None) == Q.INVALID_ARGUMENT
    assert go(struct_size=4) == Q.ABI_MISMATCH
    assert go(data_type=Q.U8) == Q.UNSUPPORTED_DATA_TYPE
    assert go(rows=0) == go(columns=0) == Q.OK
    assert go(rows=2 ** 24, columns=2 ** 11) == Q.UNSUPPORTED  # more blocks than a launch has threads for
    for bad in (dict(rows=2 ** 24 + 1), dict(columns=2 ** 20 + 1), dict(x=None), dict(codes=None), dict(scales=None), dict(x=FAKE + 1),
                dict(codes=FAKE + 2 ** 16 + 8), dict(scales=FAKE + 2 ** 17 + 2), dict(x_row_stride=511), dict(code_row_stride=504),
                dict(code_row_stride=520), dict(gated=1), dict(scale_row_stride=3), dict(scale_row_stride=0), dict(scale_block_stride=0),
                dict(scale_block_stride=5, scale_row_stride=1), dict(codes=FAKE + 16), dict(scales=FAKE + 4), dict(scales=FAKE + 2 ** 16),
                dict(row_count=FAKE + 2 ** 16), dict(row_count=FAKE + 2), dict(row_count=FAKE + 2 ** 17 + 8), dict(x_row_stride=2 ** 40)):
        assert go(**bad) == Q.INVALID_ARGUMENT, bad


PRODUCT = dict(d_type=30, a=FAKE, a_row_stride=256, a_scales=FAKE + 2 ** 16, a_scale_row_stride=2, a_scale_block_stride=1, b=FAKE + 2 ** 17,
               b_row_stride=256, b_scales=FAKE + 2 ** 18, b_scale_row_stride=2, b_scale_block_stride=1, d=FAKE + 2 ** 19, d_row_stride=64,
               m=4, n=64, k=256, d_ops__ab_scale=1.0)
BAD_PRODUCTS = (dict(m=2 ** 24 + 1), dict(n=2 ** 24 + 1), dict(k=0), dict(k=2 ** 20 + 1), dict(a=None), dict(a_scales=None), dict(b=None),
                dict(b_scales=None), dict(d=None), dict(a=FAKE + 8), dict(b=FAKE + 2 ** 17 + 4), dict(a_scales=FAKE + 2 ** 16 + 2),
                dict(b_scales=FAKE + 2 ** 18 + 1), dict(d=FAKE + 2 ** 19 + 1), dict(d_ops__bias=FAKE + 1), dict(a_row_stride=255),
                dict(a_row_stride=264), dict(b_row_stride=240), dict(a_row_stride=2 ** 24 + 16), dict(d_row_stride=63),
                dict(a_scale_row_stride=2 ** 22 + 1), dict(a_scale_block_stride=2 ** 32), dict(b_scale_row_stride=2 ** 32),
                # d meets an input
                dict(d=FAKE), dict(d=FAKE + 4 * 256 - 2), dict(d=FAKE + 2 ** 16), dict(d=FAKE + 2 ** 17 + 64 * 256 - 2), dict(d=FAKE + 2 ** 18),
                dict(d_ops__bias=FAKE + 2 ** 19 + 2))


def test_matmul_refusals():
    from stark_amd import fp8 as F, qmm as Q
    lib = Q.lib()

    def go(**kw):
        return lib.stark_qmm_fp8_matmul(C.byref(_struct(F._MatmulArgs, PRODUCT, kw)), None)

    n = C.c_uint64(77)
    assert lib.stark_qmm_fp8_matmul(None, None) == Q.INVALID_ARGUMENT
    assert lib.stark_qmm_fp8_matmul_workspace_size(None, C.byref(n)) == Q.INVALID_ARGUMENT
    assert lib.stark_qmm_fp8_matmul_workspace_size(C.byref(_struct(F._MatmulArgs, PRODUCT, {})), None) == Q.INVALID_ARGUMENT
    assert go(struct_size=4) == Q.ABI_MISMATCH
    assert go(d_type=Q.U8) == Q.UNSUPPORTED_DATA_TYPE
    assert go(d_ops__rht_factors=FAKE) == Q.UNSUPPORTED_D_OP
    assert go(m=0) == go(n=0) == go(m=0, a=None, d=None) == Q.OK
    for bad in BAD_PRODUCTS:
        assert go(**bad) == Q.INVALID_ARGUMENT, bad
    # a call in parts: 64 rows, N 4096, K 12288
    parts = dict(m=64, n=4096, k=12288, a_row_stride=12288, b_row_stride=12288, d_row_stride=4096, d=FAKE + 2 ** 28, b=FAKE + 2 ** 22,
                 a_scales=FAKE + 2 ** 21, b_scales=FAKE + 2 ** 27, a_scale_row_stride=96, b_scale_row_stride=96)
    assert lib.stark_qmm_fp8_matmul_workspace_size(C.byref(_struct(F._MatmulArgs, PRODUCT, parts)), C.byref(n)) == Q.OK
    assert n.value == 4 * 4 * 64 * 4096
    assert go(**parts) == go(**parts, workspace=FAKE + 2 ** 29 + 8, workspace_size=n.value) == Q.INVALID_ARGUMENT
    for meets in (parts["d"] + 16, FAKE, parts["b"] + 16, parts["a_scales"], parts["b_scales"] + 16):
        assert go(**parts, workspace=meets, workspace_size=n.value) == Q.INVALID_ARGUMENT
    assert go(**parts, workspace=FAKE + 2 ** 29, workspace_size=n.value - 1) == Q.WORKSPACE_TOO_SMALL
    assert lib.stark_qmm_fp8_matmul_workspace_size(C.byref(_struct(F._MatmulArgs, PRODUCT, {})), C.byref(n)) == Q.OK and n.value == 0


def test_grouped_refusals():
    from stark_amd import fp8 as F, qmm as Q
    lib = Q.lib()
    base = dict({"product__" + n: v for n, v in PRODUCT.items()}, experts=3, group_start=FAKE + 2 ** 20, b_expert_stride=64 * 256,
                b_scale_expert_stride=2)

    def make(**kw):
        s = _struct(F._GroupedArgs, base, kw)
        if "product__struct_size" not in kw:
            s.product.struct_size = C.sizeof(s.product)
        return C.byref(s)

    def go(**kw):
        return lib.stark_qmm_fp8_grouped_matmul(make(**kw), None)

    n = C.c_uint64(77)
    assert lib.stark_qmm_fp8_grouped_matmul(None, None) == Q.INVALID_ARGUMENT
    assert lib.stark_qmm_fp8_grouped_matmul_workspace_size(None, C.byref(n)) == Q.INVALID_ARGUMENT
    assert lib.stark_qmm_fp8_grouped_matmul_workspace_size(make(), None) == Q.INVALID_ARGUMENT
    assert go(struct_size=4) == go(product__struct_size=4) == Q.ABI_MISMATCH
    assert go(product__d_ops__rht_factors=FAKE) == Q.UNSUPPORTED_D_OP
    assert go(product__m=0) == go(product__n=0) == Q.OK
    for bad in [{"product__" + n: v for n, v in b.items()} for b in BAD_PRODUCTS] + [
            dict(experts=0), dict(experts=1025), dict(group_start=None), dict(group_start=FAKE + 2 ** 20 + 1), dict(b_expert_stride=8),
            dict(a_rows=FAKE + 2 ** 21, a_row_count=0), dict(a_rows=FAKE + 2 ** 21 + 2, a_row_count=9), dict(group_start=FAKE + 2 ** 19),
            dict(a_rows=FAKE + 2 ** 19 + 8, a_row_count=9), dict(product__d=FAKE + 2 ** 17 + 2 * 64 * 256),
            dict(product__d=FAKE + 8 * 256, a_rows=FAKE + 2 ** 21, a_row_count=9)]:
        assert go(**bad) == Q.INVALID_ARGUMENT, bad
    # 32-bit places of gathered rows
    assert go(a_rows=FAKE + 2 ** 21, a_row_count=2 ** 24 + 1) == Q.UNSUPPORTED
    assert go(a_rows=FAKE + 2 ** 21, a_row_count=2 ** 11, product__a_scale_row_stride=2 ** 20) == Q.UNSUPPORTED


PLAN = dict(ids=FAKE, group_start=FAKE + 2 ** 18, tokens_out=FAKE + 2 ** 19, slots=FAKE + 2 ** 20, tokens=16, active=8, experts=128)


def test_plan_refusals():
    from stark_amd import fp8 as F, qmm as Q
    lib = Q.lib()

    def go(**kw):
        return lib.stark_qmm_expert_plan(C.byref(_struct(F._PlanArgs, PLAN, kw)), None)

    n = C.c_uint64(77)
    assert lib.stark_qmm_expert_plan(None, None) == Q.INVALID_ARGUMENT
    assert lib.stark_qmm_expert_plan_workspace_size(C.byref(_struct(F._PlanArgs, PLAN, {})), C.byref(n)) == Q.OK and n.value == 0
    assert lib.stark_qmm_expert_plan_workspace_size(C.byref(_struct(F._PlanArgs, PLAN, dict(tokens=2 ** 20))), C.byref(n)) == Q.OK
    assert n.value > 0 and n.value % 16 == 0
    assert go(struct_size=4) == Q.ABI_MISMATCH
    for bad in (dict(experts=0), dict(experts=1025), dict(active=0), dict(tokens=2 ** 21 + 1), dict(ids=None), dict(group_start=None),
                dict(tokens_out=None), dict(slots=None), dict(ids=FAKE + 1), dict(group_start=FAKE + 2 ** 18 + 2), dict(slots=FAKE + 4 * 127),
                dict(tokens_out=FAKE), dict(slots=FAKE + 2 ** 19 + 8), dict(group_start=FAKE + 2 ** 19 + 4), dict(tokens=2 ** 12),
                dict(tokens=2 ** 12, workspace=FAKE + 2 ** 24 + 8, workspace_size=2 ** 20),
                dict(tokens=2 ** 12, workspace=FAKE + 2 ** 19, workspace_size=2 ** 20)):
        assert go(**bad) == Q.INVALID_ARGUMENT, bad
    assert go(tokens=2 ** 12, workspace=FAKE + 2 ** 24, workspace_size=16) == Q.WORKSPACE_TOO_SMALL


COMBINE = dict(data_type=30, x=FAKE, slots=FAKE + 2 ** 17, weights=FAKE + 2 ** 18, out=FAKE + 2 ** 20, x_row_stride=64, out_row_stride=64, tokens=8,
               active=4, rows=32, width=64)


def test_combine_refusals():
    from stark_amd import fp8 as F, qmm as Q
    call = Q.lib().stark_qmm_expert_combine

    def go(**kw):
        return call(C.byref(_struct(F._CombineArgs, COMBINE, kw)), None)

    assert call(None, None) == Q.INVALID_ARGUMENT
    assert go(struct_size=4) == Q.ABI_MISMATCH
    assert go(data_type=Q.U8) == Q.UNSUPPORTED_DATA_TYPE
    assert go(tokens=0) == go(width=0) == Q.OK
    for bad in (dict(active=0), dict(active=1025), dict(tokens=2 ** 24), dict(width=2 ** 24 + 1), dict(rows=2 ** 31), dict(x=None),
                dict(slots=None), dict(weights=None), dict(out=None), dict(x=FAKE + 1), dict(weights=FAKE + 2 ** 18 + 2), dict(x_row_stride=63),
                dict(out_row_stride=63), dict(out=FAKE), dict(out=FAKE + 2 ** 17), dict(out=FAKE + 2 ** 18 + 4)):
        assert go(**bad) == Q.INVALID_ARGUMENT, bad
