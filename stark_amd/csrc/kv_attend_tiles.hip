// Attention over the 4-bit paged key/value cache for requests of many rows: prompts, and verify of long drafts.
#include "kv_attend.h"

namespace {

using namespace qmm;

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kKeys = 64;  // keys of a tile: four records

// LDS of one tile: keys [key][value of the head], values transposed [value of the head][key], both f16 in 16-byte pieces
// whose place in a row is swizzled by the row, so that 16 lanes that read the same piece of 16 rows meet no bank twice.
// not_finite: keys (bits) whose values' planes are not finite, for each group; they stand as zeros in v.
// kLse and kFine: keys are their codes less 8, and planes holds scales and middles (the value of code 8) of the keys, [group]
// [scale or middle][key].
// kFine: values are code times the leading bits of their scale, exact, and rest holds what the two leave of a value, f16, by four
// keys: scale / leading - 1 of each, then their biases.
enum { kPlain, kLse, kFine };
template <int DIM, int G, int MODE>
struct Tile {
    static constexpr bool EXACT = MODE != kPlain, FINE = MODE == kFine;
    u32x4 k[kKeys][DIM / 8];
    u32x4 v[DIM][kKeys / 8];
    unsigned long long not_finite[G];
    alignas(16) uint32_t absent[4];  // records whose page is not in the cache
    alignas(16) float planes[EXACT ? G : 1][2][EXACT ? kKeys : 4];
    alignas(16) uint16_t rest[FINE ? G : 1][FINE ? kKeys / 4 : 1][2][4];
    static QMM_DEVICE uint32_t key_piece(uint32_t key, uint32_t piece) {
        return piece ^ (DIM >= 128 ? key & 15 : key >> 1 & 7);
    }
    static QMM_DEVICE uint32_t value_piece(uint32_t dim, uint32_t piece) { return piece ^ (dim >> 1 & 7); }
};

QMM_DEVICE f16x2 half2_of(uint32_t w) { return __builtin_bit_cast(f16x2, w); }
QMM_DEVICE uint32_t bits_of(f16x2 h) { return __builtin_bit_cast(uint32_t, h); }

// Largest of three, one instruction; a NaN wins (its row is NaN in any case).
QMM_DEVICE float max3(float a, float b, float c) {
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

// Two codes (bits 0-3 and 16-19 of w) as values: 1024 + c by its bits, less 1024 exactly, then one rounding of s c + b.
QMM_DEVICE uint32_t two_values(uint32_t w, f16x2 s, f16x2 b) {
    const f16x2 c = half2_of(and_or(w, 0x000f000fu, 0x64006400u)) - (f16x2){(_Float16)1024.0f, (_Float16)1024.0f};
    return bits_of(__builtin_elementwise_fma(c, s, b));
}

// Of two f16 scales the seven leading bits (less where that would leave a subnormal with nothing): a product with a code has
// eleven and is exact.
QMM_DEVICE uint32_t leading(uint32_t w) {
    const u16x2 h = __builtin_bit_cast(u16x2, w), low = {127, 127}, cut = __builtin_bit_cast(u16x2, w & 0xfff0fff0u);
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(cut, __builtin_elementwise_min(h, low)));
}

// Two codes less 8, exact.
QMM_DEVICE uint32_t two_codes(uint32_t w) {
    return bits_of(half2_of(and_or(w, 0x000f000fu, 0x64006400u)) - (f16x2){(_Float16)1032.0f, (_Float16)1032.0f});
}

// What one thread brings of a tile: of one record, a lane's key words and value words, and their planes.
template <int DIM, int G>
struct Codes {
    static constexpr int N = DIM / 32;  // words of a lane
    uint32_t kc[N], vc[N], kp[G];
    u32x4 vp[G];
    uint32_t own[(G + 3) / 4];  // kFine: value planes of the lane's key lane % 16, groups lane / 16 and lane / 16 + 4

    QMM_DEVICE void load_keys(const uint8_t* rec, uint32_t lane) {
        const uint32_t c = lane & 15, g = lane >> 4;
        const uint8_t* p = rec + (DIM == 64 ? c * 32 + g * 8 : c * 64 + g * 16);
        if (DIM == 64) {
            *(u32x2*)kc = *(const u32x2*)p;
        } else {
#pragma unroll
            for (int h = 0; h < DIM / 128; ++h) *(u32x4*)&kc[4 * h] = *(const u32x4*)(p + 1024 * h);
        }
#pragma unroll
        for (int gr = 0; gr < G; ++gr) kp[gr] = *(const uint32_t*)(rec + 8 * DIM + 64 * gr + 4 * c);
    }
    template <int MODE>
    QMM_DEVICE void load_values(const uint8_t* rec, uint32_t lane) {
        const uint8_t* p = rec + 8 * DIM + 64 * G + lane * (DIM == 64 ? 8 : 16);
        if (DIM == 64) {
            *(u32x2*)vc = *(const u32x2*)p;
        } else {
#pragma unroll
            for (int h = 0; h < DIM / 128; ++h) *(u32x4*)&vc[4 * h] = *(const u32x4*)(p + 1024 * h);
        }
#pragma unroll
        for (int gr = 0; gr < G; ++gr) vp[gr] = *(const u32x4*)(rec + 16 * DIM + 64 * G + 64 * gr + 16 * (lane >> 4));
        if (MODE == kFine)
#pragma unroll
            for (int j = 0; j < (G + 3) / 4; ++j)
                own[j] = *(const uint32_t*)(rec + 16 * DIM + 64 * G + 64 * ((lane >> 4) % G + 4 * j) + 4 * (lane & 15));
    }
    // record: 0 .. 3 in the tile
    template <int MODE>
    QMM_DEVICE void write_keys(Tile<DIM, G, MODE>& t, uint32_t record, uint32_t lane) const {
        constexpr bool EXACT = MODE != kPlain;
        const uint32_t key = 16 * record + (lane & 15), g = lane >> 4;
#pragma unroll
        for (int j = 0; j < N; ++j) {  // word 4 j + g: values 8 (4 j + g) .. + 7, of group j G / N
            const f16x2 plane = half2_of(kp[j * G / N]), s = {plane[0], plane[0]}, b = {plane[1], plane[1]};
            const uint32_t w = kc[j];
            t.k[key][t.key_piece(key, 4 * j + g)] =
                EXACT ? u32x4{two_codes(w), two_codes(w >> 4), two_codes(w >> 8), two_codes(w >> 12)}
                      : u32x4{two_values(w, s, b), two_values(w >> 4, s, b), two_values(w >> 8, s, b), two_values(w >> 12, s, b)};
        }
        if (EXACT) {
#pragma unroll
            for (int gr = 0; gr < G; ++gr)
                if ((int)g == gr % 4) {
                    t.planes[gr][0][key] = plane_scale(kp[gr]);
                    t.planes[gr][1][key] = plane_middle(kp[gr]);
                }
        }
    }
    // live: bit e: the lane's token 4 (lane / 16) + e is a key that some row may see, in a page of the cache
    template <int MODE>
    QMM_DEVICE void write_values(Tile<DIM, G, MODE>& t, uint32_t record, uint32_t lane, uint32_t live) {
        const uint32_t r = lane & 15, quad = lane >> 4;
        u32x4 q[G];  // (copies: the loaded registers stay as they are, or the next load's would be copied, and waited for)
#pragma unroll
        for (int gr = 0; gr < G; ++gr) q[gr] = vp[gr];
        if (__any(live != 15)) {
#pragma unroll
            for (int gr = 0; gr < G; ++gr)
#pragma unroll
                for (int e = 0; e < 4; ++e) q[gr][e] = live >> e & 1 ? q[gr][e] : 0u;
        }
        u16x2 top = {0, 0};  // largest magnitude bits
#pragma unroll
        for (int gr = 0; gr < G; ++gr)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, (uint32_t)(q[gr][e] & 0x7fff7fffu)));
        if (__any(top[0] >= 0x7c00u || top[1] >= 0x7c00u)) {
#pragma unroll
            for (int gr = 0; gr < G; ++gr)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if ((q[gr][e] & 0x7c00u) == 0x7c00u || (q[gr][e] >> 16 & 0x7c00u) == 0x7c00u) {
                        q[gr][e] = 0;
                        if (r == 0) atomicOr(&t.not_finite[gr], 1ull << (16 * record + 4 * quad + e));
                    }
        }
        if (MODE == kFine) {
#pragma unroll
            for (int j = 0; j < (G + 3) / 4; ++j) {
                const uint32_t w = own[j];
                const float all = plane_scale(w), lead = plane_scale(leading(w));
                const bool finite = (w & 0x7c00u) != 0x7c00u && (w >> 16 & 0x7c00u) != 0x7c00u;
                const float part = lead != 0.0f ? (all - lead) * __builtin_amdgcn_rcpf(lead) : 0.0f;
                if (quad < (uint32_t)G) {
                    auto& to = t.rest[MODE == kFine ? quad + 4 * j : 0][MODE == kFine ? 4 * record + r / 4 : 0];
                    to[0][r % 4] = finite ? (uint16_t)f32_to_f16_bits(part) : 0, to[1][r % 4] = finite ? (uint16_t)(w >> 16) : 0;
                }
            }
        }
        // quads 0 and 2 of a record share a piece, and 1 and 3: the order of the probabilities in their operand
        const uint32_t piece = 2 * record + (quad & 1), half = quad >> 1;
#pragma unroll
        for (int i = 0; i < DIM / 32; ++i) {  // byte i of the lane's value words: values 32 i + 2 r and the next
            constexpr int M = DIM / 32;
            const u32x4 p = q[i * G / M];
            f16x2 s01 = half2_of(permb(p[1], p[0], 0x05040100u)), b01 = half2_of(permb(p[1], p[0], 0x07060302u));
            f16x2 s23 = half2_of(permb(p[3], p[2], 0x05040100u)), b23 = half2_of(permb(p[3], p[2], 0x07060302u));
            if (MODE == kFine) {
                s01 = half2_of(leading(bits_of(s01))), s23 = half2_of(leading(bits_of(s23)));
                b01 = b23 = f16x2{(_Float16)0.0f, (_Float16)0.0f};
            }
            uint32_t w01, w23;
            if (DIM == 64) {
                const uint32_t sel = 0x0c000c00u | (uint32_t)(2 + i) << 16 | (uint32_t)i;
                w01 = permb(0, vc[0], sel), w23 = permb(0, vc[1], sel);
            } else {
                const uint32_t sel = 0x0c000c00u | (uint32_t)(4 + i % 4) << 16 | (uint32_t)(i % 4);
                const int o = i / 4 * 4;
                w01 = permb(vc[o + 1], vc[o], sel), w23 = permb(vc[o + 3], vc[o + 2], sel);
            }
            const uint32_t d = 32 * i + 2 * r;
            u32x2* lo = (u32x2*)&t.v[d][t.value_piece(d, piece)];
            u32x2* hi = (u32x2*)&t.v[d + 1][t.value_piece(d + 1, piece)];
            lo[half] = u32x2{two_values(w01, s01, b01), two_values(w23, s23, b23)};
            hi[half] = u32x2{two_values(w01 >> 4, s01, b01), two_values(w23 >> 4, s23, b23)};
        }
    }
};

// The request whose workgroups (kv::row_tiles) `id` is one of, and which of them: the last request whose first is at or
// before it, by a search of 64 at a time. 256 requests of one token (4 query heads to each of 8 key heads, 1000 keys) beside a
// prompt of 8192: 757 us, and 1081 with as many workgroups for each request as the longest has.
QMM_DEVICE bool find_request(const AttendArgs& a, uint32_t id, uint32_t lane, uint32_t* b, uint32_t* turn) {
    uint32_t from = 0, count = a.batch, first = 0;
    for (;;) {  // the request is one of count, from `from`
        const uint32_t each = (count + 63) / 64, i = lane * each;
        uint32_t mine = 0xffffffffu;
        if (i < count) {
            const int32_t start = min(max(a.query_start[from + i], 0), (int32_t)a.tokens);
            mine = (uint32_t)kv::row_tiles((uint64_t)start * a.ratio, from + i);
        }
        const uint64_t here = __ballot(mine <= id);
        if (here == 0) return false;  // before the first request
        const uint32_t n = (uint32_t)__popcll((unsigned long long)here) - 1;
        from += n * each, count = min(each, count - n * each);
        first = (uint32_t)__builtin_amdgcn_readlane((int)mine, (int)n);
        if (each == 1) break;
    }
    *b = from, *turn = id - first;
    return true;
}

// Schedule: N matrix products, each operand read from LDS four products ahead.
template <int N>
QMM_DEVICE void read_ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
}

// Prompts: tiles of 128 rows (a kv head's query heads times tokens, 32 to a wave) against tiles of 64 keys.
//
// The keys and values of a tile are made f16 values in LDS once for all four waves (2 packed operations a value); what that
// rounds, 2^-12 of a value, is of the size of the probabilities' own rounding to f16. Scores come out transposed, from
// v_mfma_f32_32x32x16_f16 with keys as rows and query rows as columns: a lane holds, of one row, 16 of each 32 keys, and
// those are the second product's B operand as they stand: the order of the keys in the transposed values is chosen to
// match. One pass over the keys, running reference of the exponents and sum; the reference moves only when a probability
// nears the end of f16, which a tile's sum shows.
// Two tiles of LDS: the next tile is unpacked while this one is multiplied, and the one after that is in flight.
// Bound by vector work beside the matrix cores: per 64 keys and 32 rows 32 products of 32x32x16 (1024 clocks) stand beside
// 32 exponentials (512 clocks) and some 285 other vector instructions (1140), of which the unpacking has 150. 2048 tokens of
// 32 heads on 8 of 128 against 4096 + 2048 keys take 207 to 224 us by the card, 256 on one (830 to 770 TFLOP/s; a large library
// product reaches 1130 to 1306). On a card where they took 213 they took 160 when the unpacking was left out for a measurement,
// 189 without the products. Slower were 256 rows to a workgroup with 8 waves (254, causal tiles of unlike length then stand
// alone on a CU) and with 64 rows to a wave (314, one wave a SIMD does not hide its own latencies); a running maximum taken from
// every tile's scores took 221, and so did the compiler's own order of LDS reads.
// kLse (bf16 with lse): the score products take the codes themselves, exact in f16, one sum a scale group, and a key's planes
// are applied to the scores in f32, as in kv_attend_rows; and lse is of the sum of the probabilities before they are rounded.
// Keys rounded to f16 move a score by up to 2^-11 of scale |q| |k|, which bf16 outputs do not show, but an f32 lse does.
// kFine (f16): that, and neither a probability nor a value is rounded to one f16, which left outputs 1.5 times as far from
// exact arithmetic as their own rounding. With s' the seven leading bits of a value's scale, so that s' c is exact, a value is
// s c + b = s' c (1 + r) + b, and sum p v = sum p' s' c + sum (p - p' + p r) s' c + sum p b: p' is the probability's f16, the
// second factor one f16 for each scale group (r is below 2^-6, so it is held to 2^-17 of p; 2^-3 and 2^-14 where a scale is
// subnormal), the third sum f32. The keys' planes cost 2 G + 1 operations a score, the values' 1.5 G + 3 and a second product:
// the same chunk takes 213, 217 and 224 us with 1, 2 and 4 groups in bf16, 240, 272 and 403 with lse, 336, 369 and 478 in f16.
template <int DIM, int G, int MODE>
__global__ __launch_bounds__(256, DIM <= 128 ? 2 : 1) void kv_attend_tiles(AttendArgs a) {
    constexpr bool EXACT = MODE != kPlain, FINE = MODE == kFine;
    constexpr int J = DIM / 16;   // k blocks of a score product
    constexpr int O = DIM / 32;   // blocks of the output
    using T = Tile<DIM, G, MODE>;
    __shared__ T tiles[2];
    const uint32_t lane = threadIdx.x & 63, col = lane & 31, hf = lane >> 5;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // workgroup: kv head first (workgroups are dealt to the XCDs in turn: a head's row tiles meet in one L2), then the
    // row tile, longest first, then the shortest of the rest (with two workgroups to a CU a long one meets a short one)
    uint32_t id = blockIdx.x;
    const uint32_t head = id % a.cache.kv_heads;
    id /= a.cache.kv_heads;
    const uint32_t part = id / a.turns;
    id -= part * a.turns;
    uint32_t b, turn;  // request, and which of its workgroups
    if (a.tiles) {
        b = id / a.tiles, turn = id - b * a.tiles;
    } else if (!find_request(a, id, lane, &b, &turn)) {
        return;
    }
    const kv::Request r = request_of(a, b);
    const uint32_t rows = (uint32_t)r.q_len * a.ratio;
    if (rows <= a.row_limit) return;
    const uint32_t mine = (rows + kv::kTileRows - 1) / kv::kTileRows;  // row tiles of this request
    if (turn >= mine) return;
    const uint32_t tile = turn < (mine + 1) / 2 ? mine - 1 - turn : turn - (mine + 1) / 2;

    const uint32_t row0 = tile * kv::kTileRows, row_end = min(row0 + kv::kTileRows, rows);
    const kv::Range top_row = kv::visible((int32_t)(row0 / a.ratio), r.q_len, r.kv_len, a.causal, a.window);
    const kv::Range last_row = kv::visible((int32_t)((row_end - 1) / a.ratio), r.q_len, r.kv_len, a.causal, a.window);
    // this workgroup's keys: its piece of those that the tile's rows see
    const int32_t begin = top_row.lo & ~(kKeys - 1);
    const int32_t piece = a.pieces > 1 ? kv::piece_keys(last_row.hi - begin, a.pieces) : 0;
    if (part && part * (uint64_t)piece >= (uint64_t)(last_row.hi - begin)) return;  // the join leaves it out as well
    const int32_t from = begin + (int32_t)part * piece, to = a.pieces > 1 ? min(last_row.hi, from + piece) : last_row.hi;
    const int32_t steps = from < to ? (to - from + kKeys - 1) / kKeys : 0;

    const uint32_t first = row0 + 32 * wave;  // this wave's rows
    const bool any_row = first < row_end;
    const uint32_t rho = first + col;
    const bool live = rho < row_end;
    const uint32_t qi = live ? rho / a.ratio : row0 / a.ratio, qh = head * a.ratio + (live ? rho - qi * a.ratio : 0);
    const uint32_t token = (uint32_t)r.first + qi;
    const kv::Range see = kv::visible((int32_t)qi, r.q_len, r.kv_len, a.causal, a.window);
    // of the wave's rows: keys that all see, and that some sees
    const kv::Range wave_top = kv::visible((int32_t)(min(first, row_end - 1) / a.ratio), r.q_len, r.kv_len, a.causal, a.window);
    const kv::Range wave_last = kv::visible((int32_t)((min(first + 32, row_end) - 1) / a.ratio), r.q_len, r.kv_len, a.causal,
                                            a.window);
    const int32_t inner_lo = __builtin_amdgcn_readfirstlane(wave_last.lo), outer_lo = __builtin_amdgcn_readfirstlane(wave_top.lo);
    const int32_t inner_hi = __builtin_amdgcn_readfirstlane(min(wave_top.hi, to));
    const int32_t outer_hi = __builtin_amdgcn_readfirstlane(any_row ? min(wave_last.hi, to) : 0);

    const uint32_t record = wave;  // that this wave unpacks of each tile
    const int32_t* table = a.table + (size_t)b * a.stride;
    const uint32_t page_mask = (1u << a.cache.page_shift) - 1;
    const uint8_t* base = a.cache.data + (uint64_t)head * a.cache.head_bytes;
    Codes<DIM, G> codes;
    const auto page_of = [&](int32_t n) {  // a tile may reach past the last key: past the table too
        const uint32_t t = (uint32_t)(from + kKeys * n) + 16 * record;
        return (uint32_t)table[min(t >> a.cache.page_shift, a.stride - 1)];
    };
    // of the codes in hand: the lane's tokens of its record that are keys, and whether the record's page is in the cache
    uint32_t live_keys = 0;
    bool in_cache = false;
    const auto fetch = [&](int32_t n, uint32_t page) {
        const uint32_t t = (uint32_t)(from + kKeys * n) + 16 * record;
        in_cache = page < a.cache.page_count;
        const uint8_t* rec = base + (uint64_t)(in_cache ? page : 0) * a.cache.page_bytes + (t & page_mask) / 16 * a.cache.record;
        codes.load_keys(rec, lane);
        codes.template load_values<MODE>(rec, lane);
        const int32_t left = r.kv_len - (int32_t)(t + 4 * (lane >> 4));
        live_keys = !in_cache || left <= 0 ? 0 : left >= 4 ? 15 : (1u << left) - 1;
    };
    const auto unpack = [&](T& t) {
        codes.template write_keys<MODE>(t, record, lane);
        codes.template write_values<MODE>(t, record, lane, live_keys);
        if (lane == 0) t.absent[record] = !in_cache;
    };
    if (threadIdx.x < 2 * G) tiles[threadIdx.x / G].not_finite[threadIdx.x % G] = 0;
    uint32_t page = 0;  // of the tile to fetch next
    if (steps) {
        fetch(0, page_of(0));
        page = page_of(min(1, steps - 1));
    }

    // B operands of the score products: lane half hf holds values 8 (2 j + hf) .. + 7 of its row, in the pieces' order
    f16x8 qb[J];
    float c1, qsum[G];
    {
        const uint16_t* p = (const uint16_t*)a.q.p + (token * a.q.token + qh * a.q.head + 8 * hf);
        u32x4 w[J];
        if (a.q.vec) {
#pragma unroll
            for (int j = 0; j < J; ++j) w[j] = *(const u32x4*)(p + 16 * j);
        } else {
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) w[j][e] = p[16 * j + 2 * e] | (uint32_t)p[16 * j + 2 * e + 1] << 16;
        }
        float x[J][8], top = 0.0f;
        widen(w, a.is_bf16, x);
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[j][e]));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        // 2^k puts the largest in [2^3, 2^4): scores of keys up to 2^15 stay far inside f32 (and rows of nothing but tiny
        // values, under a scale that leaves their scores tiny as well, as they are, so that c1 stays a normal number).
        // Sums are of the scaled values, so that they pass f32 only where the scores do.
        const int k = min(3 - (top > 0.0f && top < INFINITY ? ilogbf(top) : 0), 100 + ilogbf(a.scale));
        c1 = fminf(ldexp_f32(a.scale, -k), FLT_MAX);  // positive: the sign is q's
        float sum[G];
#pragma unroll
        for (int gr = 0; gr < G; ++gr) sum[gr] = 0.0f;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = ldexp_f32(x[j][e / 2 + 4 * (e & 1)], k) * a.sign;
                qb[j][e] = (_Float16)v;
                sum[j * G / J] += v;
            }
#pragma unroll
        for (int gr = 0; gr < G; ++gr) qsum[gr] = (sum[gr] + __shfl_xor(sum[gr], 32, 64)) * c1;
    }

    f32x16 o[O];
#pragma unroll
    for (int i = 0; i < O; ++i) o[i] = f32x16{};
    float m = kNone, l = 0.0f, le = 0.0f;  // (le: of the probabilities before rounding)
    float beta[FINE ? G : 1];              // kFine: sum p b of the lane's keys
#pragma unroll
    for (int gr = 0; gr < (FINE ? G : 1); ++gr) beta[gr] = 0.0f;
    __syncthreads();  // not_finite is clear
    if (steps) {
        // the first tile may begin before the window of its first row: what stands there may be anything by now
        const int32_t hidden = top_row.lo - (from + 16 * (int32_t)record + 4 * (int32_t)(lane >> 4));
        if (hidden > 0) live_keys = hidden >= 4 ? 0 : live_keys >> hidden << hidden;
        unpack(tiles[0]);
        fetch(min(1, steps - 1), page);
        page = page_of(min(2, steps - 1));
    }
    for (int32_t n = 0; n < steps; ++n) {
        __syncthreads();
        T& t = tiles[n & 1];
        const int32_t t0 = from + kKeys * n;
        const u32x4 out = *(const u32x4*)t.absent;
        uint64_t set = 0;
#pragma unroll
        for (int gr = 0; gr < G; ++gr) set |= t.not_finite[gr];
        const bool flags = __builtin_amdgcn_readfirstlane((int)(uint32_t)(set | set >> 32)) != 0;
        if (FINE && t0 < outer_hi && t0 + kKeys > outer_lo) {
            // 32 keys after 32, to leave registers for the operands that each scale group has of its own
#pragma unroll (DIM == 64 ? 2 : 1)
            for (int h = 0; h < 2; ++h) {
                // two sums at a time, of two groups or of the halves of one
                constexpr int PARTS = G > 1 ? G : 2, N = J / PARTS;
                f32x16 s, z;
#pragma unroll
                for (int g0 = 0; g0 < PARTS; g0 += 2) {
                    f32x16 acc[2];
#pragma unroll
                    for (int n = 0; n < 2 * N; ++n) {
                        const int part = n % 2, j = (g0 + part) * N + n / 2;
                        const uint32_t key = 32 * h + col;
                        const f16x8 k = __builtin_bit_cast(f16x8, t.k[key][t.key_piece(key, 2 * j + hf)]);
                        acc[part] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qb[j], n < 2 ? f32x16{} : acc[part], 0, 0, 0);
                    }
                    if (G == 1) acc[0] += acc[1];
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int part = 0; part < (G > 1 ? 2 : 1); ++part) {
                            const int gr = G > 1 ? g0 + part : 0;
                            const uint32_t at = 32 * h + 8 * q + 4 * hf;
                            const f32x4 scale = *(const f32x4*)&t.planes[EXACT ? gr : 0][0][EXACT ? at : 0];
                            const f32x4 mid = *(const f32x4*)&t.planes[EXACT ? gr : 0][1][EXACT ? at : 0];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int i = 4 * q + e;
                                s[i] = gr ? fmaf(scale[e], acc[part][i], s[i]) : scale[e] * acc[part][i];
                                z[i] = gr ? fmaf(mid[e], qsum[gr], z[i]) : mid[e] * qsum[0];
                            }
                        }
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = fmaf(s[i], c1, z[i]);
                if (a.cap != 0.0f) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        s[i] = a.cap <= kPlainCap ? soft_capped(s[i], a.cap) : soft_capped_exact(s[i], a.cap);
                }
                const int32_t k0 = t0 + 32 * h;
                const uint32_t out0 = h ? out[2] : out[0], out1 = h ? out[3] : out[1];
                if (k0 < inner_lo || k0 + 32 > inner_hi || (out0 | out1)) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int32_t key = k0 + 8 * (i / 4) + 4 * (int32_t)hf + i % 4;
                        s[i] = key >= see.lo && key < see.hi && key < to && !(i / 8 ? out1 : out0) ? s[i] : -INFINITY;
                    }
                }
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 16; i += 2) top = max3(top, s[i], s[i + 1]);
                // the reference moves where a probability would pass 2^15, to 2^-8 of the largest (as below)
                if (__any(top - m > 15.0f)) {
                    top = fmaxf(top, __shfl_xor(top, 32, 64));
                    const float low = top - 8.0f;
                    const float mn = fmaxf(m, top - low > 8.0f ? top : low), f = __builtin_amdgcn_exp2f(m - mn);
                    m = mn;
                    le *= f;
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) beta[gr] *= f;
#pragma unroll
                    for (int i = 0; i < O; ++i) o[i] *= f;
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {  // 16 keys
                    float p[8];
                    f16x2 first[4], left[4];  // a probability's f16, and what that leaves of it
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const float x = __builtin_amdgcn_exp2f(s[8 * k + e] - m), y = __builtin_amdgcn_exp2f(s[8 * k + e + 1] - m);
                        const f16x2 v = {(_Float16)x, (_Float16)y};
                        le += x, le += y;
                        p[e] = x, p[e + 1] = y;
                        first[e / 2] = v;
                        left[e / 2] = f16x2{(_Float16)(x - (float)v[0]), (_Float16)(y - (float)v[1])};
                    }
                    const f16x8 pf = operand(bits_of(first[0]), bits_of(first[1]), bits_of(first[2]), bits_of(first[3]));
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) {
                        uint32_t second[4];
#pragma unroll
                        for (int q = 0; q < 2; ++q) {  // four keys
                            const u32x4 w = *(const u32x4*)&t.rest[FINE ? gr : 0][FINE ? 8 * h + 4 * k + 2 * q + hf : 0];
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const f16x2 b = half2_of(w[2 + e]);
                                second[2 * q + e] = bits_of(__builtin_elementwise_fma(first[2 * q + e], half2_of(w[e]), left[2 * q + e]));
                                beta[gr] = fmaf(p[4 * q + 2 * e], (float)b[0], beta[gr]);
                                beta[gr] = fmaf(p[4 * q + 2 * e + 1], (float)b[1], beta[gr]);
                            }
                        }
                        const f16x8 ps = operand(second[0], second[1], second[2], second[3]);
                        f16x8 v[O / G];
#pragma unroll
                        for (int i = 0; i < O / G; ++i) {
                            const uint32_t d = 32 * (gr * O / G + i) + col;
                            v[i] = __builtin_bit_cast(f16x8, t.v[d][t.value_piece(d, 2 * (2 * h + k) + hf)]);
                        }
#pragma unroll
                        for (int i = 0; i < O / G; ++i)
                            o[gr * O / G + i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i], pf, o[gr * O / G + i], 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < O / G; ++i)
                            o[gr * O / G + i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i], ps, o[gr * O / G + i], 0, 0, 0);
                    }
                }
            }
        } else if (!FINE && t0 < outer_hi && t0 + kKeys > outer_lo) {
            f32x16 s[2];
            // two sums at a time, so that no product waits for the last: of both blocks of 32 keys, or of two scale groups
            constexpr int P = EXACT && G > 1 ? 2 : 1, H = 3 - P;
#pragma unroll
            for (int h0 = 0; h0 < 2; h0 += H) {
                f32x16 z;  // of the keys' middles
#pragma unroll
                for (int g0 = 0; g0 < (EXACT ? G : 1); g0 += P) {
                    constexpr int N = EXACT ? J / G * P : J;  // products of P groups
                    f32x16 acc[H][P];
#pragma unroll
                    for (int n = 0; n < N; ++n)
#pragma unroll
                        for (int h = 0; h < H; ++h) {
                            const int gr = n % P, j = (g0 + gr) * (N / P) + n / P;
                            const uint32_t key = 32 * (h0 + h) + col;
                            const f16x8 k = __builtin_bit_cast(f16x8, t.k[key][t.key_piece(key, 2 * j + hf)]);
                            acc[h][gr] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qb[j], n < P ? f32x16{} : acc[h][gr], 0, 0, 0);
                        }
                    read_ahead<N * H>();
#pragma unroll
                    for (int h = 0; h < H; ++h) {
                        if (!EXACT) {
                            s[h0 + h] = acc[h][0];
                            continue;
                        }
#pragma unroll
                        for (int q = 0; q < 4; ++q)
#pragma unroll
                            for (int gr = 0; gr < P; ++gr) {
                                const uint32_t at = 32 * (h0 + h) + 8 * q + 4 * hf;
                                const f32x4 scale = *(const f32x4*)&t.planes[EXACT ? g0 + gr : 0][0][EXACT ? at : 0];
                                const f32x4 mid = *(const f32x4*)&t.planes[EXACT ? g0 + gr : 0][1][EXACT ? at : 0];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const int i = 4 * q + e;
                                    const float v = acc[h][gr][i];
                                    s[h0 + h][i] = g0 + gr ? fmaf(scale[e], v, s[h0 + h][i]) : scale[e] * v;
                                    z[i] = g0 + gr ? fmaf(mid[e], qsum[g0 + gr], z[i]) : mid[e] * qsum[0];
                                }
                            }
                        if (g0 + P == G)
#pragma unroll
                            for (int i = 0; i < 16; ++i) s[h0 + h][i] = fmaf(s[h0 + h][i], c1, z[i]);
                    }
                }
            }
            // value i of block h: key 32 h + 8 (i / 4) + 4 hf + i % 4
            const auto cap_scores = [&](auto capped) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[h][i] = capped(EXACT ? s[h][i] : s[h][i] * c1, a.cap);
            };
            if (a.cap != 0.0f) {
                if (a.cap <= kPlainCap) cap_scores(soft_capped);
                else cap_scores(soft_capped_exact);
            }
            float scale = EXACT || a.cap != 0.0f ? 1.0f : c1;
            if (t0 < inner_lo || t0 + kKeys > inner_hi || (out[0] | out[1] | out[2] | out[3])) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const uint32_t at = 32 * h + 8 * (i / 4) + 4 * hf + i % 4;
                        const int32_t key = t0 + (int32_t)at;
                        s[h][i] = key >= see.lo && key < see.hi && key < to && !out[2 * h + i / 8] ? s[h][i] : -INFINITY;
                    }
            }
            // probabilities to f16 (2^-11 of each); the sum is of the same rounded values, which takes half the instructions
            // and leaves the average of a row unbiased
            uint32_t p[2][8];
            float sum, exact;
            const auto probabilities = [&]() {
                sum = exact = 0.0f;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float even = __builtin_amdgcn_exp2f(fmaf(s[h][2 * i], scale, -m));
                        const float odd = __builtin_amdgcn_exp2f(fmaf(s[h][2 * i + 1], scale, -m));
                        const f16x2 v = {(_Float16)even, (_Float16)odd};
                        p[h][i] = bits_of(v);
                        if (EXACT) exact += even + odd;
                        sum = __builtin_amdgcn_fdot2(v, (f16x2){(_Float16)1.0f, (_Float16)1.0f}, sum, false);
                    }
            };
            probabilities();
            // The reference of the exponents moves only when a probability is near the end of f16 (at first, from kNone, all
            // are infinite); whether one is shows in their sum. It moves to 2^-8 of the largest: probabilities keep all their
            // bits down to 2^-22 of it (15 in natural logarithms), and some down to 2^-33.
            if (__any(sum > 0x1p15f)) {
                // With scores past 2^24 s * scale - m in one rounding is not 0 where m is s * scale rounded: infinite
                // probabilities of 2^64 and more also come here, and go once both are rounded alike.
                float top = -INFINITY;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        s[h][i] *= scale, s[h][i + 1] *= scale;
                        asm("" : "+v"(s[h][i]), "+v"(s[h][i + 1]));  // (the compiler would make one rounding of it again)
                        top = max3(top, s[h][i], s[h][i + 1]);
                    }
                scale = 1.0f;
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                const float low = top - 8.0f;  // (past 2^27 this may be 16 less)
                const float mn = fmaxf(m, top - low > 8.0f ? top : low), f = __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= f, le *= f;
#pragma unroll
                for (int i = 0; i < O; ++i) o[i] *= f;
                probabilities();
            }
            l += sum, le += exact;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
#pragma unroll
                for (int i = 0; i < O; ++i) {
                    const uint32_t d = 32 * i + col;
                    const f16x8 v = __builtin_bit_cast(f16x8, t.v[d][t.value_piece(d, 2 * h + hf)]);
                    const uint32_t* q = &p[h / 2][h % 2 * 4];
                    o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, operand(q[0], q[1], q[2], q[3]), o[i], 0, 0, 0);
                }
            }
            read_ahead<4 * O>();
        }
        // values that are not finite, of keys that the row sees
        if (flags && t0 < outer_hi && t0 + kKeys > outer_lo) {
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                const uint64_t bad = t.not_finite[gr];
                const int32_t lo = min(max(see.lo - t0, 0), 64), hi = min(max(see.hi - t0, 0), 64);
                const uint64_t below_hi = hi >= 64 ? ~0ull : (1ull << hi) - 1, below_lo = lo >= 64 ? ~0ull : (1ull << lo) - 1;
                const float add = bad & below_hi & ~below_lo ? __builtin_nanf("") : 0.0f;
#pragma unroll
                for (int i = gr * O / G; i < (gr + 1) * O / G; ++i) o[i] += add;
            }
        }
        // the tile after this (past the last: the last again), and the loads of the one after that
        unpack(tiles[(n + 1) & 1]);
        fetch(min(n + 2, steps - 1), page);
        page = page_of(min(n + 3, steps - 1));
        // this tile's flags are clear again before the tile after the next sets them
        if (flags) {
            __syncthreads();
            if (threadIdx.x < G) t.not_finite[threadIdx.x] = 0;
        }
    }

    l += __shfl_xor(l, 32, 64), le += __shfl_xor(le, 32, 64);
    if (FINE) {
        l = le;
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            const float bias = beta[FINE ? gr : 0] + __shfl_xor(beta[FINE ? gr : 0], 32, 64);
#pragma unroll
            for (int i = gr * O / G; i < (gr + 1) * O / G; ++i) o[i] += bias;
        }
    }
    if (!live) return;
    const float sum = EXACT ? le : l;
    // value 4 q + e of block i: 32 i + 8 q + 4 hf + e
    // the pieces of a tile that fit one need no join
    if (a.pieces == 1 || piece >= last_row.hi - begin) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint16_t* p = (uint16_t*)a.out.p + (token * a.out.token + qh * a.out.head + 4 * hf);
#pragma unroll
        for (int i = 0; i < O; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float v[4] = {o[i][4 * q], o[i][4 * q + 1], o[i][4 * q + 2], o[i][4 * q + 3]};
                store_out<4>(p + 32 * i + 8 * q, a.out.vec, a.is_bf16, v, inv);
            }
        if (a.lse && hf == 0)
            a.lse[(size_t)token * a.heads + qh] = sum == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(sum)) * kLn2;
    } else {
        // (the join divides by the sum before rounding)
        const float f = MODE == kLse && l > 0.0f ? sum / l : 1.0f;
        const size_t at = ((size_t)token * a.heads + qh) * a.pieces + part;
        float* dst = a.tile_po + at * DIM + 4 * hf;
#pragma unroll
        for (int i = 0; i < O; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *(f32x4*)(dst + 32 * i + 8 * q) = f32x4{o[i][4 * q], o[i][4 * q + 1], o[i][4 * q + 2], o[i][4 * q + 3]} * f;
        if (hf == 0) a.tile_pml[at] = float2{sum == 0.0f ? kNone : m, sum};
    }
}

// The pieces of a row: out = sum_c o_c 2^(m_c - m) / sum_c l_c 2^(m_c - m), in the order of the pieces. DIM / 4 lanes to a
// row, four values each. Bound by the latency of its chain of reads (lengths, then statistics, then partial outputs).
template <int DIM>
__global__ __launch_bounds__(256) void kv_attend_tiles_join(AttendArgs a) {
    constexpr uint32_t L = DIM / 4;
    const uint32_t lane = threadIdx.x & 63, id = blockIdx.x * (256 / L) + threadIdx.x / L, d = threadIdx.x % L * 4;
    const uint32_t token = min(id / a.heads, a.tokens - 1), qh = id % a.heads;
    // the request of the token: the last that starts at or before it (the wave's rows may be of several tokens)
    uint32_t before = 0;
    const uint32_t low = (uint32_t)__builtin_amdgcn_readfirstlane((int)token);
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 64) {
        const uint64_t here = __ballot(b0 + lane < a.batch && a.query_start[b0 + lane] <= (int32_t)low);
        before += (uint32_t)__popcll((unsigned long long)here);
        if (~here) break;
    }
    while (before < a.batch && a.query_start[before] <= (int32_t)token) ++before;
    if (before == 0 || id / a.heads >= a.tokens) return;
    const kv::Request r = request_of(a, before - 1);
    const uint32_t rows = (uint32_t)r.q_len * a.ratio, qi = token - (uint32_t)r.first;
    if ((int32_t)token < r.first || qi >= (uint32_t)r.q_len || rows <= a.row_limit) return;
    const uint32_t row0 = (qi * a.ratio + qh % a.ratio) / kv::kTileRows * kv::kTileRows;
    // the row's tile, its keys and its pieces, as kv_attend_tiles has them
    const kv::Range top_row = kv::visible((int32_t)(row0 / a.ratio), r.q_len, r.kv_len, a.causal, a.window);
    const kv::Range last_row = kv::visible((int32_t)((min(row0 + kv::kTileRows, rows) - 1) / a.ratio), r.q_len, r.kv_len,
                                           a.causal, a.window);
    const int32_t range = last_row.hi - (top_row.lo & ~(kKeys - 1)), piece = kv::piece_keys(range, a.pieces);
    if (piece >= range) return;  // its tile wrote it
    const uint32_t parts = (uint32_t)(range + piece - 1) / (uint32_t)piece;
    const size_t base = ((size_t)token * a.heads + qh) * a.pieces;
    float m = kNone;
    for (uint32_t c = 0; c < parts; ++c) m = fmaxf(m, a.tile_pml[base + c].x);
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
#pragma unroll 4
    for (uint32_t c = 0; c < parts; ++c) {
        const float2 v = a.tile_pml[base + c];
        const float f = __builtin_amdgcn_exp2f(v.x - m);
        l = fmaf(v.y, f, l);
        sum += *(const f32x4*)(a.tile_po + (base + c) * DIM + d) * f;
    }
    const float y[4] = {sum[0], sum[1], sum[2], sum[3]};
    uint16_t* p = (uint16_t*)a.out.p + (token * a.out.token + qh * a.out.head + d);
    store_out<4>(p, a.out.vec, a.is_bf16, y, l == 0.0f ? 0.0f : 1.0f / l);
    if (a.lse && d == 0) a.lse[(size_t)token * a.heads + qh] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

template <int DIM, int G>
stark_qmm_status launch(const AttendArgs& a, hipStream_t s) {
    const uint32_t blocks = a.cache.kv_heads * a.turns * a.pieces;  // below 2^24 (kv::fits)
    if (!a.is_bf16) hipLaunchKernelGGL((kv_attend_tiles<DIM, G, kFine>), dim3(blocks), dim3(256), 0, s, a);
    else if (a.lse) hipLaunchKernelGGL((kv_attend_tiles<DIM, G, kLse>), dim3(blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((kv_attend_tiles<DIM, G, kPlain>), dim3(blocks), dim3(256), 0, s, a);
    QMM_HIP_CHECK(hipGetLastError());
    if (a.pieces > 1) {  // then the row tiles are fewer than workgroups fit the GPU
        const uint32_t each = 1024 / DIM, joins = (a.heads * a.tokens + each - 1) / each;
        hipLaunchKernelGGL((kv_attend_tiles_join<DIM>), dim3(joins), dim3(256), 0, s, a);
        QMM_HIP_CHECK(hipGetLastError());
    }
    return STARK_QMM_OK;
}

}  // namespace

namespace qmm {

stark_qmm_status launch_attend_tiles(const AttendArgs& a, hipStream_t s) {
    switch (a.cache.dim * 16 + a.cache.groups) {
    case 64 * 16 + 1: return launch<64, 1>(a, s);
    case 64 * 16 + 2: return launch<64, 2>(a, s);
    case 128 * 16 + 1: return launch<128, 1>(a, s);
    case 128 * 16 + 2: return launch<128, 2>(a, s);
    case 128 * 16 + 4: return launch<128, 4>(a, s);
    case 256 * 16 + 2: return launch<256, 2>(a, s);
    case 256 * 16 + 4: return launch<256, 4>(a, s);
    default: return launch<256, 8>(a, s);
    }
}

}  // namespace qmm
