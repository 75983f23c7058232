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

// Keys that query token i (0 .. q_len - 1) of a request sees: [lo, hi). Its position is kv_len - q_len + i.
struct Range {
    int32_t lo, hi;
};
KV_HD Range visible(int32_t i, int32_t q_len, int32_t kv_len, bool causal, uint32_t window) {
    const int64_t pos = (int64_t)kv_len - q_len + i;
    int64_t hi = causal && pos + 1 < kv_len ? pos + 1 : kv_len;
    int64_t lo = window && pos + 1 > (int64_t)window ? pos + 1 - (int64_t)window : 0;
    if (hi < 0) hi = 0;
    if (lo > hi) lo = hi;
    return {(int32_t)lo, (int32_t)hi};
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

// Rows of a tile: query rows (token i, query head h of the kv head's `ratio`) numbered i * ratio + h.
constexpr uint32_t kRows = 16;

// Keys that any row of a tile sees.
KV_HD Range tile_range(uint32_t tile, uint32_t ratio, int32_t q_len, int32_t kv_len, bool causal, uint32_t window) {
    const uint32_t last = tile * kRows + kRows - 1, rows = (uint32_t)q_len * ratio;
    const Range a = visible((int32_t)(tile * kRows / ratio), q_len, kv_len, causal, window);
    const Range b = visible((int32_t)((last < rows ? last : rows - 1) / ratio), q_len, kv_len, causal, window);
    return {a.lo, b.hi};
}

// Keys of one workgroup where `units` (requests x kv heads x row tiles) do not fill the GPU, and how many such
// chunks a request has at most. A multiple of 128, so that the four waves' 32-key steps come out even.
struct Split {
    uint32_t chunk, chunks;
};
KV_HD Split split(uint64_t units, uint32_t max_kv, uint32_t cus) {
    const uint64_t want = 4ull * cus;
    if (units >= want || max_kv <= 256) return {max_kv < 128 ? 128 : (max_kv + 127) / 128 * 128, 1};
    const uint32_t parts = (uint32_t)((want + units - 1) / units);
    uint32_t chunk = ((max_kv + parts - 1) / parts + 127) / 128 * 128;
    if (chunk < 256) chunk = 256;
    return {chunk, (max_kv + chunk - 1) / chunk};
}

}  // namespace kv
