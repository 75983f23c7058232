// Layout and index arithmetic of the 4-bit paged key/value cache. Plain functions (no HIP types), so that
// the tests run the same arithmetic on the CPU.
//
// The cache is [page][kv head][tile] of records; a record holds 16 tokens of one kv head:
//   key codes    8 * dim bytes
//   key planes   [group][16 tokens] words: f16 scale | f16 bias << 16
//   value codes  8 * dim bytes
//   value planes as the key planes
// A record is a multiple of 128 bytes, read with 16-byte loads that cover whole lines.
//
// Codes are laid out for v_mfma_f32_16x16x32_f16, into whose A operand they go from the load with a mask
// and no lane exchange:
// * Keys: A row = token, k = 32 values of the head. Code word d of a token (8 values 8d..8d+7, value n in
//   bits 4n) belongs to k block d / 4, lane group d % 4; the words of one lane (its k blocks in order, up to
//   four) are contiguous, and the 64 lanes' pieces are 512 or 1024 contiguous bytes.
// * Values: A row = 16 values of the head, k = tokens. Lane r of a 16-lane row holds, of each token, the values
//   32 i + 2 r + e (i = 0.., e = 0, 1) as nibble 2 i + e, four tokens together. All 16 rows of one product are
//   then in the same block of 32 values, so in the same scale group, and an output lane's 8 values are
//   contiguous.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define KV_HD __host__ __device__ __forceinline__
#else
#define KV_HD inline
#endif

namespace kv {

constexpr uint32_t kTile = 16;      // tokens of a record
constexpr float kLimit = 32768.0f;  // largest magnitude a group holds (its values fit f16 after rounding)

KV_HD uint32_t codes_bytes(uint32_t dim) { return 8u * dim; }
KV_HD uint32_t planes_bytes(uint32_t groups) { return 64u * groups; }
KV_HD uint32_t record_bytes(uint32_t dim, uint32_t groups) { return 2u * (codes_bytes(dim) + planes_bytes(groups)); }

// Byte of key code word d (0 .. dim / 8 - 1) of token t (0 .. 15), from the start of the key codes.
KV_HD uint32_t key_word(uint32_t dim, uint32_t t, uint32_t d) {
    const uint32_t row = dim < 128 ? dim / 8 : 16;  // words of a token in one 1024-byte (dim 64: 512-byte) block
    return (d / row) * 1024u + t * row * 4u + (d % 4u) * row + (d % row) / 4u * 4u;
}

// Byte of value byte i (values 128 half + 32 i + 2 r and the next) of lane r, token t, from the start of the
// value codes. dim 64: half 0, i = 0, 1; else i = 0 .. 3.
KV_HD uint32_t value_byte(uint32_t dim, uint32_t t, uint32_t half, uint32_t r, uint32_t i) {
    const uint32_t w = dim < 128 ? 2u : 4u;  // bytes a token holds for one lane
    return half * 1024u + (t / 4u * 16u + r) * 4u * w + (t % 4u) * w + i;
}

KV_HD uint32_t plane_word(uint32_t t, uint32_t group) { return (group * 16u + t) * 4u; }

// Record of token position `at` (inside its page) of a page and head.
KV_HD uint64_t record_index(uint64_t page, uint32_t kv_heads, uint32_t head, uint32_t page_size, uint32_t at) {
    return (page * kv_heads + head) * (page_size / kTile) + at / kTile;
}

// Keys that query token i (0 .. q_len - 1) of a request sees: [lo, hi). Its position is kv_len - q_len + i, so none sees
// past kv_len; the position may be before the first key. window: 0, or below 2^31.
struct Range {
    int32_t lo, hi;
};
KV_HD Range visible(int32_t i, int32_t q_len, int32_t kv_len, bool causal, int32_t window) {
    const int32_t end = kv_len - q_len + i + 1;  // at most kv_len
    int32_t hi = causal ? end : kv_len, lo = window && end > window ? end - window : 0;
    hi = hi < 0 ? 0 : hi;
    lo = lo > hi ? hi : lo;
    return {lo, hi};
}

// A request of an attention call, with lengths that no device value can push past what was checked.
struct Request {
    int32_t first, q_len, kv_len;  // first query row, query rows, keys
};
KV_HD Request request(int32_t start, int32_t end, int32_t kv_len, uint32_t tokens, uint32_t max_query, uint32_t max_kv) {
    const int32_t n = (int32_t)tokens;
    const int32_t a = start < 0 ? 0 : start > n ? n : start, e = end < a ? a : end > n ? n : end;
    const int32_t q = e - a > (int32_t)max_query ? (int32_t)max_query : e - a;
    const int32_t k = kv_len < 0 ? 0 : kv_len > (int32_t)max_kv ? (int32_t)max_kv : kv_len;
    return {a, q, k};
}

// Rows that a thread of the append does, one after another, with one read of their rotation: as many as leave 2^18 threads or
// more (4 waves a SIMD, which is what its registers leave room for), so one below 2^19 rows' threads, and up to eight.
KV_HD uint32_t rows_each(uint64_t threads) {
    const uint64_t each = threads / (1u << 18);
    return each < 1 ? 1 : each > 8 ? 8 : (uint32_t)each;
}

// Plan of one request: pages it holds before and after the step, of at most `width`.
struct PagePlan {
    int32_t before, need;
};
KV_HD PagePlan page_plan(int64_t cached, int64_t added, uint32_t page_shift, uint32_t width) {
    const int64_t round = ((int64_t)1 << page_shift) - 1;
    int64_t before = (cached + round) >> page_shift, after = (cached + added + round) >> page_shift;
    if (before > width) before = width;
    if (after > width) after = width;
    return {(int32_t)before, (int32_t)(after - before)};
}

// Keys that any row of a request sees (its q_len is not 0).
KV_HD Range request_range(int32_t q_len, int32_t kv_len, bool causal, int32_t window) {
    return {visible(0, q_len, kv_len, causal, window).lo, visible(q_len - 1, q_len, kv_len, causal, window).hi};
}

// Requests that the decode kernel takes in a call: those of up to `limit` rows (a kv head's query heads times new tokens),
// in blocks of `block` rows (8 or 16). Where the bounds say that no request has more than 64 rows it takes all (16 requests
// of 16 to 40 rows and 900 to 9000 keys 27 us with it, 50 in tiles, 64 of them 64 and 135; where many requests have 64 rows
// and one length tiles are up to 1.4 times faster, 64 of 2000 keys 127 and 90); in a call of longer requests those of one
// block, which has what one new token has (decode rows among prompts), where there may be enough of them to pay for two more
// launches, else none (0). The others go to the tile kernel. Us with them and without: beside a prompt of 300, 2 decode rows of
// 2000 keys 58 and 46, 8 58 and 50, 16 65 and 57, 64 106 and 125; beside one of 100, 8 of 200 keys 27 and 19, 16 of 300 29 and 21,
// 64 of 300 32 and 35, 16 of 8000 119 and 121. (So 16 requests are few: tiles won ground there when their workgroups came to be
// counted by rows.)
struct Rows {
    uint32_t limit, block;
};
KV_HD Rows row_limit(uint32_t batch, uint32_t max_query, uint32_t ratio, uint32_t max_kv) {
    const uint64_t most = (uint64_t)max_query * ratio;
    if (most <= 64) return {64, most <= 8 ? 8u : 16u};
    if (ratio > 16 || (batch < 16 && (uint64_t)batch * max_kv < 49152) || batch == 1) return {0, 16};
    const uint32_t block = ratio <= 8 ? 8 : 16;
    return {block, block};
}

// Keys of a workgroup's least share of a decode call: two steps for each of its four waves.
constexpr uint32_t kLeastKeys = 256;

// What beginning a unit costs a workgroup, in keys: its steps are counted as so many more. Blocks of 8 rows, us with 512,
// 1024 and 2048: 16 requests of 900 to 9000 keys 24.9, 23.2 and 24.8; 64 of 500 to 32768 132, 128.4 and 136; 256 of 100 to 2100
// 68, 67.5 and 75. Blocks of 16, whose keys take longer: 16 requests of 900 to 9000 keys and 16 to 40 rows 26.6 with 512, 28.7
// with 1024.
KV_HD uint32_t unit_keys(uint32_t block) { return block == 8 ? 1024 : 512; }

// Steps of each of `grid` workgroups that share `total` (below 2^31): a multiple of four, one for each wave.
// inverse: 2^32 / grid, rounded down (2^32 - 1 for 1).
KV_HD uint32_t share_of(uint32_t total, uint32_t grid, uint32_t inverse, uint32_t step_keys) {
    uint32_t per = (uint32_t)((uint64_t)total * inverse >> 32);
    while (per * grid < total) ++per;  // the quotient was up to two short
    per = (per + 3) / 4 * 4;
    const uint32_t least = kLeastKeys / step_keys;
    return per < least ? least : per;
}

// How a decode call's work is dealt: whole units (a request's rows on one kv head) to a workgroup where no unit has more
// than 1024 keys, or 2048 with 128 units; else `grid` workgroups share all steps (no more workgroups than shares). Us, whole
// and shared, 8 kv heads: 8 requests of 1000 keys 12.6 and 15.2, 64 of 100 to 1000 16.2 and 23.8, 16 of 100 to 2000 14.8 and
// 16.1, 64 of them 20.6 and 24.5; one of 2000 keys 19.2 and 12.0, 64 of 100 to 4000 34.7 and 30.9.
struct Share {
    uint32_t whole, grid;
};
KV_HD Share share(uint32_t batch, uint32_t kv_heads, uint32_t block, uint32_t max_kv, uint32_t slots) {
    if (max_kv <= 1024 || (max_kv <= 2048 && (uint64_t)batch * kv_heads >= 128)) return {1, 0};
    const uint64_t keys = (uint64_t)batch * kv_heads * (max_kv + 128ull + unit_keys(block)), most = (keys + kLeastKeys - 1) / kLeastKeys;
    return {0, most < slots ? (uint32_t)(most ? most : 1) : slots};
}

// Least keys of a piece of a row tile's keys.
constexpr int32_t kPieceKeys = 256;

// Keys of each of up to `pieces` pieces of a range: a multiple of 64, so that all pieces but the last are alike.
KV_HD int32_t piece_keys(int32_t range, uint32_t pieces) {
    const int64_t each = (((int64_t)range + pieces - 1) / pieces + 63) / 64 * 64;
    return (int32_t)(each < kPieceKeys ? kPieceKeys : each > 0x7fffffc0 ? 0x7fffffc0 : each);
}

constexpr uint32_t kTileRows = 128;  // of the tile kernel

// Workgroups for row tiles on a kv head, by the query rows of all requests: request b's first is row_tiles of the rows before
// it and b. Up to the next request's there is room for its tiles, and at most one workgroup more.
KV_HD uint64_t row_tiles(uint64_t rows, uint32_t requests) { return rows / kTileRows + requests; }

// Row tiles of the tile kernel: how many a request has at most, and how many pieces the keys of a tile are cut into where
// the tiles do not fill the GPU (two workgroups to a CU). 512 tokens of 32 heads on 8 against 5120 keys: 75.7 us in 4
// pieces, 85.0 in 8, with 7 of partial outputs less. `rows` is what the call's query rows come to on one kv head.
struct Tiling {
    uint32_t tiles, pieces;
};
KV_HD Tiling tiling(uint32_t batch, uint32_t kv_heads, uint64_t rows, uint64_t most_rows, uint32_t max_kv, uint32_t cus) {
    const uint64_t have = kv_heads * row_tiles(rows, batch), want = (2ull * cus + have - 1) / have;
    const uint64_t longest = ((uint64_t)max_kv + kPieceKeys - 1) / kPieceKeys;
    return {(uint32_t)((most_rows + kTileRows - 1) / kTileRows), (uint32_t)(want < longest ? want : longest ? longest : 1)};
}

// Whether the launches of a call stay inside what is counted: workgroups in 24 bits and shared steps in 31. blocks: of rows in
// the decode kernel (0: it takes none); rows: of the call on a kv head, where some are the tile kernel's, else 0. (Pieces add
// less than two workgroups a CU.)
KV_HD bool fits(uint32_t batch, uint32_t kv_heads, uint32_t blocks, uint32_t max_kv, uint64_t rows) {
    const uint64_t units = (uint64_t)batch * kv_heads * blocks;
    const bool whole = share(batch, kv_heads * blocks, 16, max_kv, 1).whole;
    if (blocks && (whole ? units >= 1ull << 24 : units * (max_kv / 32 + 40ull) >= 1ull << 31)) return false;
    return !rows || kv_heads * row_tiles(rows, batch) < (1ull << 24) - (1u << 17);
}

}  // namespace kv
