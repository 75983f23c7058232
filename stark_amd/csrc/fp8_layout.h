// Plain arithmetic of the 8-bit floating-point products, for the host, the device and CPU tests.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define FP8_BOTH __host__ __device__ inline
#else
#define FP8_BOTH inline
#endif

namespace fp8 {

constexpr uint32_t kBlock = 128;  // values to a scale, on both axes

FP8_BOTH uint32_t blocks(uint32_t n) { return (n + kBlock - 1) / kBlock; }

// Rows of one group, from the starts as the caller's memory has them.
struct Range {
    uint32_t first, count;
};
FP8_BOTH Range group(int32_t start, int32_t end, uint32_t rows) {
    const uint32_t lo = start < 0 ? 0 : (uint32_t)start < rows ? (uint32_t)start : rows;
    const uint32_t hi = end < 0 ? 0 : (uint32_t)end < rows ? (uint32_t)end : rows;
    return {lo, hi > lo ? hi - lo : 0};
}

// Row tiles that groups of `rows` rows in all need at most: each group with rows has one that is not full.
FP8_BOTH uint32_t row_tiles(uint32_t rows, uint32_t groups, uint32_t tile) {
    return groups == 1 ? (rows + tile - 1) / tile : rows / tile + (groups < rows ? groups : rows);
}

// Tile of the i-th workgroup, which runs on XCD i % 8: each XCD takes a run of consecutive tiles, whose
// operands then share its L2. Not below `tiles`: this workgroup has none.
FP8_BOTH uint32_t tile_of(uint32_t i, uint32_t tiles) {
    const uint32_t per = (tiles + 7) / 8, local = i >> 3;
    return local < per ? (i & 7) * per + local : tiles;
}

// Place of a tile among row tiles and column tiles: bands of eight row tiles, in a band a column of tiles after the other, so
// that the tiles that run at once on an XCD (32) share eight row tiles' and four column tiles' operands.
struct Place {
    uint32_t row, column;  // row: not below `rows` where there is no such tile
};
FP8_BOTH Place place(uint32_t i, uint32_t rows, uint32_t columns) {
    constexpr uint32_t kBand = 8;
    if (i >= rows * columns) return {rows, 0};
    const uint32_t band = i / (kBand * columns), in = i - band * kBand * columns, left = rows - band * kBand;
    const uint32_t high = left < kBand ? left : kBand;
    return {band * kBand + in % high, in / high};
}

// Whether tiles of 256 x 256 pay, against 128 x 128: they read half the operands, and need rows and tiles enough.
FP8_BOTH bool wide_tiles(uint32_t rows, uint32_t groups, uint32_t n) {
    return rows / groups >= 256 && (uint64_t)row_tiles(rows, groups, 256) * ((n + 255) / 256) >= 192;
}

// Strips of 16 columns and waves of a workgroup of the few-rows kernel. Some eight waves a CU are enough loads in flight; more
// only shorten their runs, and a run of less than four blocks is mostly its own start (N 12288, K 4096, one row: 4 waves 10.6 us,
// 8 waves 14.4, 16 waves 20.9; N 4096, K 12288, five rows: 8 waves 12.9, 16 waves 15.8). With strips for every CU several
// times over, two strips share a row's codes and a start (128 experts of N 1536, K 2048, one or two rows each: 2 strips and 4
// waves 43.3 us, 1 and 2 44.4, 1 and 4 57.5).
struct RowShare {
    uint32_t strips, waves;
};
FP8_BOTH RowShare row_share(uint64_t row_tiles, uint32_t n, uint32_t k) {
    const uint64_t units = row_tiles * ((n + 15) / 16);
    if (units >= 4096) return {2, 4};
    uint32_t waves = 2;
    while (waves < 16 && units * waves < 2048 && waves < blocks(k)) waves *= 2;
    return {1, waves};
}

// item / blocks by the inverse floor(2^32 / blocks) (0xffffffff for 1): the estimate is at most one short.
struct Split {
    uint32_t row, block;
};
FP8_BOTH Split split(uint32_t item, uint32_t blocks, uint32_t inverse) {
    uint32_t q = (uint32_t)(((uint64_t)item * inverse) >> 32), r = item - q * blocks;
    if (r >= blocks) q += 1, r -= blocks;
    return {q, r};
}
FP8_BOTH uint32_t inverse(uint32_t blocks) { return blocks > 1 ? (uint32_t)((1ull << 32) / blocks) : 0xffffffffu; }

}  // namespace fp8
