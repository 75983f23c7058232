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

// Strips of 16 columns and waves of a workgroup of the few-rows kernel. Some eight waves a CU are enough loads in flight; more
// only shorten their runs, and a run of less than eight blocks is mostly its own start (N 12288, K 4096, one row: 4 waves 10.6
// us, 8 waves 14.4, 16 waves 20.9; N 4096, K 4096, 16 rows: 4 waves 7.4, 8 waves 8.3; N 4096, K 12288, five rows: 8 waves 12.9,
// 16 waves 15.8). With strips for every CU several
// times over, two strips share a row's codes and a start (128 experts of N 1536, K 2048, one or two rows each: 2 strips and 4
// waves 43.3 us, 1 and 2 44.4, 1 and 4 57.5).
struct RowShare {
    uint32_t strips, waves;
};
FP8_BOTH RowShare row_share(uint64_t row_tiles, uint32_t n, uint32_t k) {
    const uint64_t units = row_tiles * ((n + 15) / 16);
    if (units >= 4096) return {2, 4};
    uint32_t waves = 2;
    while (waves < 16 && units * waves < 2048 && waves * 8 < blocks(k)) waves *= 2;
    return {1, waves};
}

// Which kernel takes a product, by what it would take in microseconds. Each form's time is a start and the larger of its steps one
// after the other and its work at the rate that it reaches; each was fitted to calls of 16 to 4096 rows, N 1001 to 12288, K 2000
// to 12288, and experts of 1 to 512 rows on average, and is within some 20% of them where it is the least. Measured on both sides
// of where it changes (us): 32 rows, N 12288, K 4096: few rows 20.8, tiles of 64 15.0. 64 rows, N = K = 4096: few rows 11.8, tiles
// of 64 15.4, in four parts 11.3. 128 rows, N 1001, K 2000: few rows 6.2, tiles of 64 12.5. 512 rows, N 4096, K 4096: tiles of 64
// 17.8, of 128 26.2; 1024 rows 32.6 and 27.1. 64 rows, N 4096, K 12288: four parts 16.1, one 40.2. 128 experts, N 1536, K 2048: 64
// tokens (4 rows an expert): few rows 64.8, tiles of 64 73.6; 256 tokens 108 and 83.4; 2048 tokens: tiles of 128 137, of 256 149;
// 8192 tokens 350 and 308.
struct Choice {
    uint32_t tile;   // 64, 128 or 256; 0: the few-rows kernel, of `rows` rows (16 or 32) a workgroup
    uint32_t rows;
    uint32_t parts;  // of the inner axis (tiles of a product without groups only)
};
FP8_BOTH Choice choose(uint32_t m, uint32_t n, uint32_t k, uint32_t groups, bool grouped, bool exact) {
    const float used = (float)(groups < m ? groups : m), each = (float)m / used;  // groups with rows, rows of one
    const float steps = (float)blocks(k), fk = (float)k, fn = (float)n;
    const auto tiles = [&](float rows) {  // row tiles: half of a group's last one is empty
        const float full = (float)m / rows + (grouped ? used / 2 : 0.0f);
        return grouped ? (full > used ? full : used) : (float)((m + (uint32_t)rows - 1) / (uint32_t)rows);
    };
    const float weights = used * fn * fk / 5.5e6f;  // once from memory
    Choice best{0, 16, 1};
    float least = 3.4e38f;
    const auto offer = [&](float us, Choice c) {
        if (us < least) least = us, best = c;
    };
    // few rows: every workgroup reads its columns' and its rows' codes
    for (uint32_t rows = 16; rows <= 32; rows *= 2) {
        if (rows == 32 && each <= (grouped ? 8.0f : 16.0f)) break;
        const float columns = rows == 16 && tiles(16) * ((n + 15) / 16) < 4096 ? 16.0f : 32.0f, groups_of = tiles((float)rows) * ((fn + columns - 1) / columns);
        const float read = ((each < rows ? each : (float)rows) + columns) * fk;  // of one workgroup
        const float all = groups_of * read / 7.8e6f, one = read / 4e4f;
        offer(3.5f + (all > one ? all : one), {0, rows, 1});
    }
    if (k < kBlock) return best;
    const struct { uint32_t tile; float start, step, work; } forms[] = {
        {64, 4.0f, exact ? 0.5f : 0.35f, exact ? 1.3e-3f : 9.5e-4f},
        {128, 5.0f, exact ? 1.08f : 0.65f, exact ? 3.6e-3f : 2.3e-3f},
        {256, 6.0f, 1.8f, 7.4e-3f}};
    for (const auto& f : forms) {
        if (f.tile == 256 && exact) continue;
        const float count = tiles((float)f.tile) * (float)((n + f.tile - 1) / f.tile);
        for (uint32_t parts = 1; parts <= (grouped || f.tile == 256 ? 1u : 8u); parts *= 2) {
            if (parts > 1 && parts * 4 > blocks(k)) break;  // four steps a part
            float us = f.step * (float)((blocks(k) + parts - 1) / parts);
            if (us < count * steps * f.work) us = count * steps * f.work;
            if (us < weights) us = weights;
            offer(f.start + us + (parts > 1 ? 3.0f + 8.0f * parts * (float)m * fn / 1e7f : 0.0f), {f.tile, 0, parts});
        }
    }
    return best;
}

// Workgroups of a call's product (without those of the join), and how many a call may have: 32 bits count them. No call whose m * n
// is at most 2^40 has more.
constexpr uint64_t kMostGroups = (1ull << 32) - 8;
FP8_BOTH uint64_t workgroups(Choice c, uint32_t m, uint32_t n, uint32_t k, uint32_t groups) {
    const uint32_t rows = row_tiles(m, groups, c.tile ? c.tile : c.rows);
    const uint32_t columns = c.tile ? c.tile : c.rows == 32 ? 32 : 16 * row_share(rows, n, k).strips;
    return (uint64_t)rows * ((n + columns - 1) / columns);
}

// A launch holds fewer than 2^32 threads; a call of more workgroups is several launches of whole eights of them.
FP8_BOTH uint32_t launch_groups(uint32_t threads) { return 0xffffffffu / threads / 8 * 8; }

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
