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
