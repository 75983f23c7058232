"""Which workgroup of the prompt kernel has which row tile (csrc/kv_layout.h, compiled for the CPU), and which calls are
more than the kernels' launches count."""
import ctypes as C
import functools
import os
import random
import subprocess
import tempfile

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stark_amd", "csrc")

_WRAP = """
#include "kv_layout.h"
extern "C" {
uint64_t row_tiles(uint64_t rows, uint32_t requests) { return kv::row_tiles(rows, requests); }
int fits(uint32_t batch, uint32_t heads, uint32_t blocks, uint32_t kv, uint64_t rows) { return kv::fits(batch, heads, blocks, kv, rows); }
}
"""


@functools.lru_cache(None)
def rules():
    with tempfile.TemporaryDirectory() as d:
        src, lib = os.path.join(d, "kv.cpp"), os.path.join(d, "kv.so")
        with open(src, "w") as f:
            f.write(_WRAP)
        subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", CSRC, src, "-o", lib], check=True)
        r = C.CDLL(lib)
        r.row_tiles.restype, r.row_tiles.argtypes = C.c_uint64, [C.c_uint64, C.c_uint32]
        r.fits.argtypes = [C.c_uint32] * 4 + [C.c_uint64]
        return r


def test_every_row_tile_has_one_workgroup():
    """Request b's workgroups begin at row_tiles(rows before it, b): there is room for its tiles before the next one's, and
    for at most one workgroup more."""
    r = random.Random(1)
    for _ in range(300):
        batch, ratio = r.randint(1, 90), r.choice([1, 2, 4, 5, 7, 16, 33])
        lengths = [r.choice([0, 1, 1, 5, r.randint(0, 700)]) for _ in range(batch)]
        before = r.choice([0, 0, 3, 200])  # rows ahead of the first request
        start = [before]
        for n in lengths:
            start.append(start[-1] + n)
        tokens = start[-1] + r.choice([0, 1, 300])
        first = [rules().row_tiles(s * ratio, b) for b, s in enumerate(start)]
        for b, n in enumerate(lengths):
            tiles = -(-n * ratio // 128)
            assert tiles <= first[b + 1] - first[b] <= tiles + 1
        assert first[-1] <= rules().row_tiles(tokens * ratio, batch)


def test_workgroups_follow_the_rows_not_the_longest_request():
    assert rules().row_tiles(2048 * 4, 1) == 65
    assert rules().row_tiles((8192 + 256) * 4, 257) == 264 + 257     # 257 requests of up to 256 tiles would be 65792
    assert rules().row_tiles((16384 + 4095) * 4, 4096) == 639 + 4096  # 2^21
    assert rules().row_tiles(2 ** 24 * 64, 2 ** 20) == 2 ** 23 + 2 ** 20


def test_calls_that_the_launches_can_count():
    fits = rules().fits
    for whole in ((2 ** 20, 16, 1, 1024, 0), (2 ** 20, 8, 2, 64, 0), (2 ** 18, 32, 2, 2048, 0)):  # a workgroup a unit
        assert not fits(*whole) and fits(whole[0] - 1, *whole[1:])
    limit = 131072 - 40 * 32  # 2^19 units of (limit / 32 + 40) = 2^12 steps
    assert not fits(2 ** 16, 8, 1, limit, 0) and fits(2 ** 16, 8, 1, limit - 1, 0)
    rows = 128 * (2 ** 21 - 2 ** 14 - 1)  # one request, 8 heads: 2^24 - 2^17 workgroups
    assert fits(1, 8, 0, 4096, rows) == 0 and fits(1, 8, 0, 4096, rows - 128) == 1
    assert fits(4096, 8, 1, 1024, 16384 * 4) and fits(1024, 8, 1, 131072, 8192 * 4)


def test_what_passes_them_is_refused_before_any_launch():
    """By the size query and by the call alike, neither of which has a GPU here."""
    from stark_amd import kv as K, qmm as Q
    for kvh, heads, batch, tokens, most, width in ((16, 16, 2 ** 20, 2 ** 20, 1, 8), (8, 32, 2 ** 16, 2 ** 16, 1, 2 ** 14),
                                                   (8, 128, 1, 2 ** 24, 2 ** 24, 8), (8, 128, 40, 2 ** 24, 2 ** 24, 8)):
        s = K._AttentionArgs()
        s.struct_size, s.cache, s.data_type = C.sizeof(s), K._Cache(1 << 20, 1 << 40, 10, 64, kvh, 128, 64), Q.BF16
        s.q = s.block_table = s.query_start = s.kv_lengths = s.workspace = 1 << 20
        s.out, s.workspace_size = 1 << 30, 1 << 40
        s.batch, s.tokens, s.heads, s.table_stride, s.max_query, s.max_kv = batch, tokens, heads, width, most, width * 64
        s.q_token_stride = s.out_token_stride = heads * 128
        s.q_head_stride = s.out_head_stride = 128
        s.scale = 0.1
        n = C.c_uint64()
        assert Q.lib().stark_qmm_kv_attention_workspace_size(C.byref(s), C.byref(n)) == Q.UNSUPPORTED
        assert Q.lib().stark_qmm_kv_attention(C.byref(s), None) == Q.UNSUPPORTED
