"""Which workgroup of the prompt kernel has which row tile (csrc/kv_layout.h, compiled for the CPU)."""
import ctypes as C
import functools
import os
import random
import subprocess
import tempfile

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stark_amd", "csrc")

_WRAP = """
#include "kv_layout.h"
extern "C" uint64_t row_tiles(uint64_t rows, uint32_t requests) { return kv::row_tiles(rows, requests); }
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
