"""The rules that choose a kernel (csrc/fp8_layout.h, compiled for the CPU) against the forms that the GPU tests name."""
import ctypes as C
import functools
import os
import random
import subprocess
import tempfile

import pytest

from tests import fp8_forms as K
from tests.test_fp8_layout import CSRC, PRODUCT, QUANTIZE, _choose, _pair, _struct, rules


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


_COUNT = """
#include "fp8_layout.h"
extern "C" uint64_t workgroups(uint32_t m, uint32_t n, uint32_t k, uint32_t groups, int grouped, int exact) {
    return fp8::workgroups(fp8::choose(m, n, k, groups, grouped, exact), m, n, k, groups);
}
extern "C" uint32_t launch_groups(uint32_t threads) { return fp8::launch_groups(threads); }
"""


@functools.lru_cache(None)
def _counts():
    with tempfile.TemporaryDirectory() as d:
        src, lib = os.path.join(d, "count.cpp"), os.path.join(d, "count.so")
        with open(src, "w") as f:
            f.write(_COUNT)
        subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", CSRC, src, "-o", lib], check=True)
        L = C.CDLL(lib)
        L.workgroups.restype = C.c_uint64
        return L


def test_launches_hold_every_call():
    """Workgroups of a call of at most 2^40 outputs are counted by 32 bits, those of a launch have fewer than 2^32 threads, and the
    sums of parts one thread for four."""
    L, r = _counts(), random.Random(2)
    sizes = [(2 ** 22, 4096, 64, 1, False), (2 ** 24, 2 ** 16, 100, 1, False), (2 ** 16, 2 ** 24, 1, 1024, True), (2 ** 20, 2 ** 20, 2 ** 20, 1, False)]
    while len(sizes) < 3000:
        m, n, k = (int(2 ** r.uniform(0, e)) for e in (24, 24, 20))
        grouped = r.random() < 0.5
        if m * n <= 2 ** 40:
            sizes.append((m, n, k, int(2 ** r.uniform(0, 10)) if grouped else 1, grouped))
    for m, n, k, groups, grouped in sizes:
        for exact in (False, True):
            assert 0 < L.workgroups(m, n, k, groups, int(grouped), int(exact)) <= 2 ** 32 - 8
            parts = _choose(m, n, k, groups, grouped, exact)[2]
            assert parts == 1 or m * -(-n // 4) + 255 < 2 ** 32
    for threads in (128, 256, 512, 1024):
        each = L.launch_groups(threads)
        assert each % 8 == 0 and 2 ** 32 - 16 * threads < each * threads < 2 ** 32


def test_calls_of_too_many_workgroups_are_refused():
    """By the size query too."""
    from stark_amd import fp8 as P, qmm as Q
    lib, n = Q.lib(), C.c_uint64(77)
    size = dict(m=2 ** 24, n=2 ** 24, d_row_stride=2 ** 24)
    call = C.byref(_struct(P._MatmulArgs, PRODUCT, size))
    assert lib.stark_qmm_fp8_matmul_workspace_size(call, C.byref(n)) == lib.stark_qmm_fp8_matmul(call, None) == Q.UNSUPPORTED
    # 34 GB of outputs in the few-rows kernel: more threads than a launch holds
    ok = C.byref(_struct(P._MatmulArgs, PRODUCT, dict(m=2 ** 22, n=4096, k=64, d_row_stride=4096)))
    assert lib.stark_qmm_fp8_matmul_workspace_size(ok, C.byref(n)) == Q.OK and n.value == 0


def test_a_quantizer_launch_holds_its_blocks():
    """2^28 - 1 blocks have 2^32 threads in whole workgroups."""
    from stark_amd import fp8 as P, qmm as Q

    def go(rows, columns):
        return Q.lib().stark_qmm_fp8_quantize(C.byref(_struct(P._QuantizeArgs, QUANTIZE, dict(rows=rows, columns=columns, x=None))), None)

    assert 49155 * 5461 == 2 ** 28 - 1 and 2 ** 12 * (2 ** 16 - 1) < 2 ** 28 - 16
    assert go(49155, 5461 * 128) == Q.UNSUPPORTED
    assert go(2 ** 16 - 1, 2 ** 12 * 128) == Q.INVALID_ARGUMENT  # no x


def test_row_shares_are_the_kernels_there_are():
    """Two strips with four waves, one with 2, 4, 8 or 16."""
    r, L = random.Random(7), rules()
    L.row_share.argtypes = [C.c_uint64, C.c_uint32, C.c_uint32, C.c_void_p]
    seen = {_pair(L.row_share, int(2 ** r.uniform(0, 20)), int(2 ** r.uniform(0, 24)), int(2 ** r.uniform(0, 20))) for _ in range(20000)}
    assert seen == {(2, 4), (1, 2), (1, 4), (1, 8), (1, 16)}


@pytest.mark.parametrize("exact", [False, True])
def test_calls_named_by_their_kernel(exact):
    for size, want in K.ROWS + K.PARTS:
        assert form(*size, exact=exact) == want
    for sizes, n, k, want in K.GROUPED:
        assert form(sum(sizes) + K.AROUND, n, k, len(sizes), True, exact) == held(want, exact)
    for tokens, active, _, experts, n, k, want in K.SHARES:
        assert form(tokens * active, n, k, experts, True, exact) == held(want, exact)
    for size, want in K.CUT_TILES:  # one group of all rows
        assert form(*size, 1, True, exact) == held(want, exact)
