// Attention over the 4-bit paged key/value cache for requests of few rows: decode and short verify.
#include "kv_attend.h"

namespace {

using namespace qmm;

// Records of a step and how they are packed. PACK (1 or 2): records whose scores share one 16 x 16 block.
template <int PACK>
struct Shape {
    static constexpr int R = 16 / PACK;            // rows of a request
    static constexpr int T = 2;                    // records of a step
    static constexpr int KEYS = 16 * T;            // keys of a step
    static constexpr int B = T / PACK;             // score blocks of a step
};

// The keys of a step of one kv head as a wave's loads leave them: code words, and of the planes each word in one lane
// only (lane 32 i + 16 v + t of pair h: record 2 h + i, keys' planes (v = 0) or values', token t).
// STREAM: loads that leave the caches to others, for blocks of 8 rows, of which a head has one: no other workgroup reads the same
// codes (us with and without, 64 requests of 4000 keys and 4 rows 58 and 66). A head's blocks of 16 rows may be several and share
// them (64 of 16 to 40 rows and 900 to 9000 keys 62 and 57, 16 of 32 rows 40.2 and 37.5). Where they turn out to be one, as the
// call's bound does not say, both sides win by turns (16 requests of 12 rows 27.1 and 25.6, 64 of them 67 and 70).
template <int DIM, int G, int T, bool STREAM>
struct Step {
    uint32_t kc[T][DIM / 32], vc[T][DIM / 32], plane[T / 2][G];
    uint32_t absent;  // bit i: record i's page is not in the cache

    // base: the head's first record in page 0; page: the records' page ids; t0: first key
    QMM_DEVICE void load(const KvCache& cache, const uint8_t* base, const uint32_t (&page)[T], uint32_t t0, uint32_t lane) {
        const uint32_t c = lane & 15, g = lane >> 4, mask = (1u << cache.page_shift) - 1;
        uint64_t rec[T];  // the records' offsets from base
        absent = 0;
#pragma unroll
        for (int i = 0; i < T; ++i) {
            const bool out = page[i] >= cache.page_count;
            absent |= out ? 1u << i : 0u;
            rec[i] = (uint64_t)(out ? 0 : page[i]) * cache.page_bytes + ((t0 + 16 * i) & mask) / 16 * cache.record;
            const uint8_t* kq = base + rec[i] + (DIM == 64 ? c * 32 + g * 8 : c * 64 + g * 16);
            const uint8_t* vq = base + rec[i] + 8 * DIM + 64 * G + lane * (DIM == 64 ? 8 : 16);
            if (DIM == 64) {
                *(u32x2*)&kc[i][0] = STREAM ? __builtin_nontemporal_load((const u32x2*)kq) : *(const u32x2*)kq;
                *(u32x2*)&vc[i][0] = STREAM ? __builtin_nontemporal_load((const u32x2*)vq) : *(const u32x2*)vq;
            } else {
#pragma unroll
                for (int h = 0; h < DIM / 128; ++h) {
                    *(u32x4*)&kc[i][4 * h] = STREAM ? load_stream(kq + 1024 * h) : *(const u32x4*)(kq + 1024 * h);
                    *(u32x4*)&vc[i][4 * h] = STREAM ? load_stream(vq + 1024 * h) : *(const u32x4*)(vq + 1024 * h);
                }
            }
        }
#pragma unroll
        for (int h = 0; h < T / 2; ++h) {
            const uint64_t even = rec[2 * h], odd = rec[2 * h + 1];
            const uint8_t* p = base + (lane & 32 ? odd : even) + (lane & 16 ? 16 * DIM + 64 * G : 8 * DIM) + 4 * c;
#pragma unroll
            for (int gr = 0; gr < G; ++gr) plane[h][gr] = *(const uint32_t*)(p + 64 * gr);
        }
    }
};

// A wave's planes of one step in LDS, [record][key or value][group][scale or middle][token] in f32: each word is
// converted once, and the 16 lanes that need the same four tokens' read them with one 16-byte read.
template <int G, int T>
struct PlaneBuffer {
    float v[T][2][G][2][16];
};

// Page ids of a wave's records: lane T n + i holds that of record i of step base + n, 64 / T steps to a load, and a step
// reads its own with v_readlane.
template <int T>
struct PageIds {
    const int32_t* row;
    uint32_t from;         // first key of step 0
    uint32_t stride;       // keys from a wave's step to its next
    uint32_t shift, last;  // last entry of the table row
    uint32_t ids, base;

    QMM_DEVICE void fill(uint32_t n, uint32_t lane) {
        base = n;
        const uint32_t t = from + stride * (n + lane / T) + 16 * (lane % T);
        ids = (uint32_t)row[min(t >> shift, last)];  // steps past the last key may be past the table too
        asm volatile("" : "+v"(ids));  // the wait for it is here, not before every v_readlane (for all loads in flight)
    }
    QMM_DEVICE void get(uint32_t n, uint32_t lane, uint32_t (&page)[T]) {
        if (n - base >= 64 / T) fill(n, lane);
#pragma unroll
        for (int i = 0; i < T; ++i) page[i] = (uint32_t)__builtin_amdgcn_readlane((int)ids, (int)(T * (n - base)) + i);
    }
};

// Running state of 16 columns: lane (c, g) holds column c.
template <int DIM, int G>
struct Running {
    static constexpr int J = DIM / 32;
    f32x4 o[2 * J];          // [32-value block, parity]: codes times p s 2^exponent, values 32 i + 2 (4 g + e) + parity
    f32x4 rounded[G];        // 8 sum p s, of the same roundings
    float beta[G], l, m;     // sum p (b + 8 s) and sum p over the lane's keys; reference of the exponents

    QMM_DEVICE void start() {
        m = kNone, l = 0.0f;
#pragma unroll
        for (int j = 0; j < 2 * J; ++j) o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int gr = 0; gr < G; ++gr) beta[gr] = 0.0f, rounded[gr] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
};

// A unit of work: one block of R rows of a request on a kv head, over the request's keys.
struct Unit {
    kv::Request r;
    kv::Range span;  // keys that some row sees
    int32_t from;    // span.lo, aligned to a step
    uint32_t rows;   // of the request on a kv head
    uint32_t steps;
    uint32_t cost;   // steps, and what a unit costs to begin
    uint32_t all;    // cost of the request's blocks on all kv heads
};

// steps: at least one where there are rows (they are written in any case); 0 (and no cost) without rows, or with too many.
template <int KEYS, int R>
QMM_DEVICE Unit unit_of(const AttendArgs& a, const kv::Request& r) {
    Unit u;
    u.r = r;
    u.rows = (uint32_t)r.q_len * a.ratio;
    u.span = kv::request_range(r.q_len, r.kv_len, a.causal, a.window);
    u.from = u.span.lo & ~(KEYS - 1);
    u.steps = (uint32_t)max((u.span.hi - u.from + KEYS - 1) / KEYS, 1);
    if (u.rows == 0 || u.rows > a.row_limit) u.steps = 0;
    u.cost = u.steps ? u.steps + kv::unit_keys(R) / KEYS : 0;
    u.all = u.cost * ((u.rows + R - 1) / R) * a.cache.kv_heads;
    return u;
}

// Lengths of 64 requests, one to a lane of the wave, so that a wave finds its way through the batch without LDS,
// barriers or a second read.
template <int KEYS, int R>
struct Requests {
    kv::Request mine;
    uint32_t b0;

    QMM_DEVICE void load(const AttendArgs& a, uint32_t first, uint32_t lane) {
        b0 = first;
        mine = {0, 0, 0};
        if (b0 + lane < a.batch) mine = request_of(a, b0 + lane);
    }
    QMM_DEVICE uint32_t cost(const AttendArgs& a) const { return unit_of<KEYS, R>(a, mine).all; }
    QMM_DEVICE Unit unit(const AttendArgs& a, uint32_t b, uint32_t lane) {
        if (b - b0 >= 64) load(a, b & ~63u, lane);
        const int l = (int)(b - b0);
        return unit_of<KEYS, R>(a, kv::Request{__builtin_amdgcn_readlane(mine.first, l),
                                               __builtin_amdgcn_readlane(mine.q_len, l),
                                               __builtin_amdgcn_readlane(mine.kv_len, l)});
    }
};

// Inclusive sum over the lanes of a wave.
template <int CTRL, int ROWS>
QMM_DEVICE uint32_t shifted(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
QMM_DEVICE uint32_t wave_scan(uint32_t v) {
    v += shifted<0x111, 0xf>(v);  // one, two, four and eight lanes to the right inside rows of 16
    v += shifted<0x112, 0xf>(v);
    v += shifted<0x114, 0xf>(v);
    v += shifted<0x118, 0xf>(v);
    v += shifted<0x142, 0xa>(v);  // the last lane of rows 0 and 2 to rows 1 and 3
    v += shifted<0x143, 0xc>(v);  // lane 31 to rows 2 and 3
    return v;
}

// Decode and verify: requests of few rows (a kv head's query heads times the new tokens), in blocks of R = 16 / PACK.
//
// The work of a call is the steps (32 keys) of all (request, kv head, block) units, in that order; each workgroup takes
// an equal run of them, so unlike lengths leave no CU idle and a workgroup pays its start once or twice, not once a
// chunk. A unit inside one run is finished there; of the others each workgroup leaves partial results, which
// kv_attend_join adds. Within a run the steps of a unit are dealt to four waves, each with its own running maximum and
// sums, joined in LDS.
//
// Keys and values stay codes. With C the codes less 8,
//   q . k = sum over groups (s_g C_g . q + (b_g + 8 s_g) sum q),   out = sum over tokens (p s_g) C + sum p (b_g + 8 s_g),
// so a key's planes are a few fma per score and group, a value's scale goes into the probability (f16, the scales times a
// power of two that keeps p s_g in f16's normal range where p s_g is 2^-22 of the wave's largest s_g or more), and a code becomes
// an f16 operand by a mask: the bits of c in the low (or 4 bits higher) end of an f16 are the subnormal c 2^-24 (c 2^-20). The 8
// is taken off by the score accumulator's start value, and for the outputs by 8 sum (p s_g), summed as it was rounded: f32 sums
// and f16 roundings then stand beside codes of either sign instead of 0 .. 15 (2.7 times less rounding error).
//
// Scores come out transposed (A rows = 16 keys, B columns = query rows): a lane holds four keys of one column in each
// block, which is the B operand of the second product as it stands, with no lane exchange. With few rows most of a
// block's 16 columns would be idle, and with them most of the vector work (planes, exponentials): so PACK records share a
// block. Record i's product takes a B operand with the rows in columns R i .. R i + R - 1 and zeros elsewhere, and all
// add into one block; column R i + r is then row r against record i's keys, and the columns of one row are joined at the
// end like the waves. In the second product each record's columns are the others' zeros.
// q is scaled per row by a power of two into f16's range, exact but for values 2^-24 below the row's largest.
//
// Bound by HBM where there are many long requests: 64 of 500 to 32768 keys, 32 heads on 8 of 128 (781 MB), take 128.5 us,
// 6.08 TB/s (a pure read of the same size 6.2). Bound by its own latency where there are few: one of 4096 keys (4.7 MB) takes
// 9.4 us and 3.9 to join; of a workgroup's 8.5 us with 64 keys 3.3 are the chain of lengths, page ids, codes and queries, 3.2
// a step and its wait, 2.0 the joining of the waves (a wave alone on its SIMD issues an instruction in 6 to 8 clocks). Blocks
// of 4 rows (four records to a score block) took 134 us there, blocks of 16 for 4 rows 67 us against 60 (64 requests of 4096
// keys); more workgroups, loads three and four steps ahead and more waves a SIMD were no faster.
//
// MODE: what the call's outputs show. Sums of products of subnormal codes lose what is below some 2^-17 of the largest product
// (measured; as if products were aligned by their factors' exponent fields): scores are off by 2e-6 to 1e-5 (root mean square,
// scores of 2), 20 to 75 times what f32 sums leave.
// kPlain (bf16 without lse): that, and one rounding of p s to f16, stand beside outputs that are rounded to 2^-9: 1.01 times
// as far from exact arithmetic as a rounding alone.
// kLse (bf16 with lse): codes of keys are made f16 numbers, c - 8, which takes one packed operation for two of them; scores
// are then as f32 sums give them (1e-7). 64 sequences 137 us, 129 without; 16 of 16 to 40 rows 26.6, 25.
// kFine (f16): values' codes as well, and p s as two f16, the second what the first leaves (2^-22 of it): an output is off by
// its own rounding, where one f16 made it 1.3 to 1.4 times as much. 64 sequences 155 us, 16 of 16 to 40 rows 29.9.
enum { kPlain, kLse, kFine };

// Two codes less 8 (bits 0-3 and 16-19 of w, or 4 bits higher and sixteenfold): 1024 + c by its bits, less 1032, exact.
QMM_DEVICE uint32_t less_8(uint32_t w) {
    const f16x2 c = __builtin_bit_cast(f16x2, and_or(w, 0x000f000fu, 0x64006400u));
    return __builtin_bit_cast(uint32_t, c - (f16x2){(_Float16)1032.0f, (_Float16)1032.0f});
}
QMM_DEVICE uint32_t less_8_sixteenfold(uint32_t w) {
    const f16x2 c = __builtin_bit_cast(f16x2, and_or(w, 0x00f000f0u, 0x64006400u));
    return __builtin_bit_cast(uint32_t, c - (f16x2){(_Float16)1152.0f, (_Float16)1152.0f});
}

template <int DIM, int G, int PACK, int MODE>
__global__ __launch_bounds__(256, DIM == 256 ? 1 : 2) void kv_attend_rows(AttendArgs a) {
    using S = Shape<PACK>;
    using Codes = Step<DIM, G, S::T, PACK == 2>;
    constexpr int R = S::R, T = S::T, KEYS = S::KEYS, B = S::B;
    constexpr int J = DIM / 32;       // k blocks of a score product, and 32-value blocks of the output
    constexpr int JG = J / G;         // of one scale group
    constexpr int kRow = DIM + 4;     // padded row of the joining buffers, floats
    __shared__ union {
        u32x4 q[J + 1][64];           // score products' B operands; the last row is zeros
        float join[4][R * kRow];
    } sh;
    __shared__ PlaneBuffer<G, T> plane_buffers[4];
    __shared__ float wave_ref[4][16], wave_sum_l[4][16];
    const uint32_t lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, row = c % R, pack = c / R;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // this workgroup's run of steps [at, end), and the request and step in it where the run begins; all steps of a
    // call are below 2^31
    uint32_t at = 0, end, per = 0, b = 0, offset;
    Requests<KEYS, R> batch;
    if (a.whole) {  // a unit to a workgroup
        const uint32_t blocks = (a.row_limit + R - 1) / R * a.cache.kv_heads;
        b = blockIdx.x / blocks;
        batch.load(a, b & ~63u, lane);
        const Unit u = batch.unit(a, b, lane);
        offset = (blockIdx.x - b * blocks) * u.cost;
        if (offset >= u.all) return;
        end = u.cost;
    } else {
        uint32_t total = 0, cost = 0, sum = 0;
        for (uint32_t b0 = 0; b0 < a.batch; b0 += 64) {
            batch.load(a, b0, lane);
            cost = batch.cost(a);
            sum = wave_scan(cost);
            total += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
        }
        per = kv::share_of(total, a.grid, a.inverse, KEYS);
        at = min(blockIdx.x * per, total), end = min(at + per, total);
        if (threadIdx.x == 0) a.begun[blockIdx.x] = int4{-1, 0, 0, 0};
        if (at == end) return;
        uint32_t done = 0;
        for (uint32_t b0 = 0;; b0 += 64) {  // at < total: some lane of some pass has it
            if (a.batch > 64) {  // else the pass above was this one
                batch.load(a, b0, lane);
                cost = batch.cost(a);
                sum = wave_scan(cost);
            }
            const uint32_t before = done + sum - cost;
            const uint64_t here = __ballot(at >= before && at - before < cost);
            if (here) {
                const int l = __ffsll((unsigned long long)here) - 1;
                b = b0 + (uint32_t)l;
                offset = at - (uint32_t)__builtin_amdgcn_readlane((int)before, l);
                break;
            }
            done += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
        }
    }
    if (threadIdx.x < 64) sh.q[J][threadIdx.x] = u32x4{0, 0, 0, 0};

    while (at < end) {
        Unit u;
        for (;; ++b, offset = 0) {  // at < total: a later request has steps
            u = batch.unit(a, b, lane);
            if (offset < u.all) break;
        }
        const uint32_t index = offset / u.cost, o0 = offset - index * u.cost, taken = min(u.cost - o0, end - at);
        // a kv head's blocks of rows one after another: they meet in the caches
        const uint32_t blocks = (u.rows + R - 1) / R, head = index / blocks, row0 = (index - head * blocks) * R;
        // a unit's first steps are its cost to begin: no work
        const uint32_t idle = u.cost - u.steps, s0 = max(o0, idle) - idle, s1 = max(o0 + taken, idle) - idle;
        const uint32_t unit_end = at + u.cost - o0;  // where the unit ends in the call's steps
        offset += taken;
        at += taken;
        if (s0 == s1) continue;

        const bool live = row0 + row < u.rows;
        const uint32_t qi = live ? (row0 + row) * a.ratio_inverse >> 16 : 0;
        const uint32_t qh = head * a.ratio + (live ? row0 + row - qi * a.ratio : 0), token = (uint32_t)u.r.first + qi;
        kv::Range see = kv::visible((int32_t)qi, u.r.q_len, u.r.kv_len, a.causal, a.window);
        if (!live) see = {0, 0x7fffffff};
        const int32_t from = u.from + KEYS * (int32_t)s0;
        const int32_t to = min(u.span.hi, u.from + KEYS * (int32_t)s1);

        // loads of the query rows (a row past the last reads the request's first one, as zeros), then the page ids and
        // the first step, and only then the use of the query rows
        u32x4 w[J];
        {
            const uint16_t* p = (const uint16_t*)a.q.p + (token * a.q.token + qh * a.q.head + 8 * g);
            if (a.q.vec) {
#pragma unroll
                for (int j = 0; j < J; ++j) w[j] = *(const u32x4*)(p + 32 * j);
            } else {
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[j][e] = p[32 * j + 2 * e] | (uint32_t)p[32 * j + 2 * e + 1] << 16;
            }
        }
        // this wave's steps: s0 + wave, s0 + wave + 4, ...
        const uint32_t steps = s0 + wave < s1 ? (s1 - s0 - wave + 3) / 4 : 0, mine = (uint32_t)from + KEYS * wave;
        PageIds<T> pages{a.table + (size_t)b * a.stride, mine, 4 * KEYS, a.cache.page_shift, a.stride - 1, 0, 0};
        const uint8_t* base = a.cache.data + (uint64_t)head * a.cache.head_bytes;
        const auto load = [&](Codes& st, uint32_t n) {
            uint32_t page[T];
            pages.get(n, lane, page);
            st.load(a.cache, base, page, mine + 4 * KEYS * n, lane);
        };
        Codes st[2];
        if (steps) {
            pages.fill(0, lane);
            load(st[0], 0);
        }

        // B operands of the score products: lane group g holds dims 8 (4 j + g) .. + 7, in the order of the code pairs
        float qsum[G], c1;
        f32x4 less8[G];
        {
            float x[J][8], top = 0.0f;
            widen(w, a.is_bf16, x);
#pragma unroll
            for (int j = 0; j < J; ++j) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[j][e] *= a.sign;
                    top = fmaxf(top, fabsf(x[j][e]));
                }
            }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            // 2^k puts the largest in [2^13, 2^14). Sums are of the scaled values, and the keys' scales bring the codes' 2^-24
            // back: no factor passes f32 where the scores do not. (The least of f32's largest: 0 stays 0 under any scale.)
            const int k = live ? 13 - (top > 0.0f && top < INFINITY ? ilogbf(top) : 0) : 0;
            c1 = fminf(ldexp_f32(a.scale, -k), FLT_MAX);
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                float s = 0.0f;
#pragma unroll
                for (int j = gr * JG; j < (gr + 1) * JG; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        x[j][e] = ldexp_f32(x[j][e], k);
                        s += x[j][e];
                    }
                s += __shfl_xor(s, 16, 64);
                s += __shfl_xor(s, 32, 64);
                s = live ? s : 0.0f;
                qsum[gr] = s * c1;
                const float v = MODE == kPlain ? s * -0x1p-21f : 0.0f;  // -8 sum q, in the accumulator's scale
                less8[gr] = f32x4{v, v, v, v};
            }
            // every wave has the same rows: wave w writes the blocks w, w + 4, ...
#pragma unroll
            for (int j = 0; j < J; ++j) {
                // code pairs of a word: nibbles (0, 4), (1, 5) sixteenfold, (2, 6), (3, 7) sixteenfold
                f16x8 h;
#pragma unroll
                for (int e = 0; e < 8; ++e) h[e] = (_Float16)(x[j][e / 2 + 4 * (e & 1)] * ((e / 2) & 1 ? 0.0625f : 1.0f));
                const u32x4 bits = __builtin_bit_cast(u32x4, h);
                if (j % 4 == (int)wave) sh.q[j][lane] = live ? bits : u32x4{0, 0, 0, 0};
            }
        }
        __syncthreads();
        // record i's operand: the rows where this lane's column is of record i, zeros elsewhere
        const auto q_operand = [&](int i, int j) {
            const u32x4* p = PACK == 1 ? &sh.q[j][lane] : &sh.q[(int)pack == i % PACK ? j : J][lane];
            return __builtin_bit_cast(f16x8, *p);
        };

        // keys that every row sees: [inner_lo, inner_hi)
        const int32_t inner_lo = kv::visible(u.r.q_len - 1, u.r.q_len, u.r.kv_len, a.causal, a.window).lo;
        const int32_t inner_hi = min(kv::visible(0, u.r.q_len, u.r.kv_len, a.causal, a.window).hi, to);

        Running<DIM, G> run;
        run.start();
        PlaneBuffer<G, T>& planes = plane_buffers[wave];
        // largest value scale (f16 bits) of plane words of a record's keys that some row sees; t: this lane's key
        const auto scale_max = [&](const uint32_t (&plane)[G], int32_t t, bool ok, uint32_t smax) {
            if ((lane & 16) && t >= u.span.lo && t < to && ok) {
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    const uint32_t h = plane[gr] & 0xffffu;
                    if (h < 0x7c00u) smax = max(smax, h);
                }
            }
            return smax;
        };
        const int32_t t_lane = (int32_t)mine + 16 * (int32_t)(lane >> 5) + (int32_t)c;  // of step 0's first plane words
        const auto wave_max = [&](uint32_t smax) {
            smax = group_max<16>(smax);
            smax = max(smax, (uint32_t)__shfl_xor((int)smax, 16, 64));
            return max(smax, (uint32_t)__shfl_xor((int)smax, 32, 64));
        };
        // On the scales of the lane's plane words: what the keys' codes are short of (c 2^-24 where they are subnormals), and the
        // values' power of two. (Not on the probabilities: the reference less an exponent would be rounded where scores pass 2^24.)
        int value_exponent = 0;
        float plane_factor = MODE == kPlain ? 0x1p24f : 1.0f;
        const auto step = [&](Codes& st, uint32_t n) {
            const int32_t t0 = (int32_t)(mine + 4 * KEYS * n);
#pragma unroll
            for (int h = 0; h < T / 2; ++h)
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    float* p = &planes.v[2 * h + (lane >> 5)][(lane >> 4) & 1][gr][0][c];
                    p[0] = plane_scale(st.plane[h][gr]) * plane_factor;
                    p[16] = plane_middle(st.plane[h][gr]);
                }
            // the reads are of other lanes' words: a wave's LDS operations run in order, and this keeps the compiler's too
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            // block u holds records PACK u .. PACK u + PACK - 1; this lane's is PACK u + pack
            float x[B][4];
#pragma unroll
            for (int u = 0; u < B; ++u) {
                f32x4 acc[G];
                // operands are read from LDS two products ahead (13.5 us with one sequence of 4096 keys; 13.9 in the
                // compiler's order, which waits for each)
                f16x8 q[3];
                q[0] = q_operand(0, 0), q[1] = q_operand(0, 1);
#pragma unroll
                for (int n = 0; n < PACK * J; ++n) {
                    const int i = n / J, j = n % J;
                    if (n + 2 < PACK * J) q[(n + 2) % 3] = q_operand((n + 2) / J, (n + 2) % J);
                    const uint32_t w = st.kc[PACK * u + i][j], v = w >> 8;
                    const f16x8 k = MODE == kPlain
                                        ? operand(w & 0x000f000fu, w & 0x00f000f0u, v & 0x000f000fu, v & 0x00f000f0u)
                                        : operand(less_8(w), less_8_sixteenfold(w), less_8(v), less_8_sixteenfold(v));
                    acc[j / JG] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        k, q[n % 3], i == 0 && j % JG == 0 ? less8[j / JG] : acc[j / JG], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
                f32x4 y, z;
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    const float* p = &planes.v[PACK * u + (PACK == 1 ? 0 : pack)][0][gr][0][4 * g];
                    const f32x4 s = *(const f32x4*)p, mid = *(const f32x4*)(p + 16);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        y[e] = gr ? fmaf(s[e], acc[gr][e], y[e]) : s[e] * acc[gr][e];
                        z[e] = gr ? fmaf(mid[e], qsum[gr], z[e]) : mid[e] * qsum[gr];
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) x[u][e] = fmaf(y[e], c1, z[e]);
            }
            if (a.cap != 0.0f) {
#pragma unroll
                for (int u = 0; u < B; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        x[u][e] = a.cap <= kPlainCap ? soft_capped(x[u][e], a.cap) : soft_capped_exact(x[u][e], a.cap);
            }
            const bool masked = t0 < inner_lo || t0 + KEYS > inner_hi || st.absent;
            if (masked) {
#pragma unroll
                for (int u = 0; u < B; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t rec = PACK * u + pack;
                        const int32_t t = t0 + 16 * (int32_t)rec + 4 * (int32_t)g + e;
                        x[u][e] = t >= see.lo && t < see.hi && t < to && !(st.absent >> rec & 1) ? x[u][e] : -INFINITY;
                    }
            }
            float top = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3]));
            if (B == 2) top = fmaxf(top, fmaxf(fmaxf(x[B - 1][0], x[B - 1][1]), fmaxf(x[B - 1][2], x[B - 1][3])));
            // the reference moves only when a score passes it by 2^6: rescaling is then rare (the difference is exact; a
            // reference of 2^26 plus 6 would be 8 more)
            if (__any(top - run.m > 6.0f)) {
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                const float mn = fmaxf(run.m, top), f = __builtin_amdgcn_exp2f(run.m - mn);
                run.m = mn;
                run.l *= f;
#pragma unroll
                for (int gr = 0; gr < G; ++gr) run.beta[gr] *= f, run.rounded[gr] *= f;
#pragma unroll
                for (int j = 0; j < 2 * J; ++j) run.o[j] *= f;
            }
            // p s to f16, half a unit of 2^-11 (kFine: and the rest): the codes it multiplies are exact
            u32x2 ps[B][G], rest[B][G];
#pragma unroll
            for (int u = 0; u < B; ++u) {
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[e] = __builtin_amdgcn_exp2f(x[u][e] - run.m);
                    run.l += p[e];
                }
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    const float* q = &planes.v[PACK * u + (PACK == 1 ? 0 : pack)][1][gr][0][4 * g];
                    f32x4 s = *(const f32x4*)q, mid = *(const f32x4*)(q + 16);
                    if (masked) {
                        // nothing of a key that a row does not see gets through, be it not a number
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool none = x[u][e] == -INFINITY;
                            s[e] = none ? 0.0f : s[e];
                            mid[e] = none ? 0.0f : mid[e];
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) run.beta[gr] = fmaf(p[e], mid[e], run.beta[gr]);
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        const float v = p[e] * s[e], w = p[e + 1] * s[e + 1];
                        const f16x2 h = {(_Float16)v, (_Float16)w};
                        ps[u][gr][e / 2] = __builtin_bit_cast(uint32_t, h);
                        if (MODE == kFine)
                            rest[u][gr][e / 2] =
                                __builtin_bit_cast(uint32_t, f16x2{(_Float16)(v - (float)h[0]), (_Float16)(w - (float)h[1])});
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // before the next step's planes are written
            const f16x8 eights = operand(0x00080008u, 0x00080008u, 0x00080008u, 0x00080008u);  // 8 2^-24
#pragma unroll
            for (int h = 0; h < T / 2; ++h) {  // records 2 h and 2 h + 1
                f16x8 pb[G], pr[G];
                const auto p_operand = [&](const u32x2 (&w)[B][G], int gr) {
                    if (PACK == 1) return operand(w[0][gr][0], w[0][gr][1], w[B - 1][gr][0], w[B - 1][gr][1]);
                    const bool lo = (int)pack == 2 * h, hi = (int)pack == 2 * h + 1;
                    return operand(lo ? w[0][gr][0] : 0, lo ? w[0][gr][1] : 0, hi ? w[0][gr][0] : 0, hi ? w[0][gr][1] : 0);
                };
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    pb[gr] = p_operand(ps, gr);
                    if (MODE == kFine) pr[gr] = p_operand(rest, gr);
                    else run.rounded[gr] = __builtin_amdgcn_mfma_f32_16x16x32_f16(eights, pb[gr], run.rounded[gr], 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < J; ++i) {  // 32-value blocks; byte i of a lane's value words
                    uint32_t w[4];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint32_t* v = st.vc[2 * h + u];
                        if (DIM == 64) {
                            const uint32_t sel = 0x0c000c00u | (uint32_t)(2 + i) << 16 | (uint32_t)i;
                            w[2 * u] = permb(0, v[0], sel);
                            w[2 * u + 1] = permb(0, v[1], sel);
                        } else {
                            const uint32_t sel = 0x0c000c00u | (uint32_t)(4 + i % 4) << 16 | (uint32_t)(i % 4);
                            v += i / 4 * 4;
                            w[2 * u] = permb(v[1], v[0], sel);
                            w[2 * u + 1] = permb(v[3], v[2], sel);
                        }
                    }
                    f16x8 lo, hi;
                    if (MODE == kFine) {
                        lo = operand(less_8(w[0]), less_8(w[1]), less_8(w[2]), less_8(w[3]));
                        hi = operand(less_8_sixteenfold(w[0]), less_8_sixteenfold(w[1]), less_8_sixteenfold(w[2]),
                                     less_8_sixteenfold(w[3]));
                    } else {
                        lo = operand(w[0] & 0x000f000fu, w[1] & 0x000f000fu, w[2] & 0x000f000fu, w[3] & 0x000f000fu);
                        hi = operand(w[0] & 0x00f000f0u, w[1] & 0x00f000f0u, w[2] & 0x00f000f0u, w[3] & 0x00f000f0u);
                    }
                    run.o[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, pb[i / JG], run.o[2 * i], 0, 0, 0);
                    run.o[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, pb[i / JG], run.o[2 * i + 1], 0, 0, 0);
                    if (MODE == kFine) {
                        run.o[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, pr[i / JG], run.o[2 * i], 0, 0, 0);
                        run.o[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, pr[i / JG], run.o[2 * i + 1], 0, 0, 0);
                    }
                }
            }
        };

        // Power of two on the values' scales: p s below 2^15 while p < 2^6, taken from the scales of the wave's first
        // records. Should a later scale be far larger, the products overflow to infinity, which shows in the sums at the
        // end: then the wave starts again with the largest scale of all its keys. Scales of 0 in the first records (zeros)
        // say nothing of the others: the wave looks at all at once.
        for (int attempt = 0; attempt < 2 && steps; ++attempt) {
            uint32_t smax = 0;
            if (attempt) {
                for (uint32_t n = 0; n < steps * (T / 2); ++n) {
                    const int32_t t = t_lane + 4 * KEYS * (int32_t)(n / (T / 2)) + 32 * (int32_t)(n % (T / 2));
                    const uint32_t id = (uint32_t)pages.row[min((uint32_t)t >> a.cache.page_shift, pages.last)];
                    const bool ok = id < a.cache.page_count;
                    const uint8_t* p = base + (uint64_t)(ok ? id : 0) * a.cache.page_bytes + 16 * DIM + 64 * G + 4 * c +
                                       ((uint32_t)t & ((1u << a.cache.page_shift) - 1)) / 16 * a.cache.record;
                    uint32_t plane[G];
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) plane[gr] = *(const uint32_t*)(p + 64 * gr);
                    smax = scale_max(plane, t, ok, smax);
                }
                pages.fill(0, lane);
                load(st[0], 0);
            } else {
                smax = scale_max(st[0].plane[0], t_lane, !(st[0].absent >> (lane >> 5) & 1), 0);
            }
            smax = wave_max(smax);
            if (smax == 0 && attempt == 0) continue;
            run.start();
            value_exponent = smax ? 8 - ilogbf(f16_bits_to_f32(smax)) : 0;
            if (lane & 16) plane_factor = ldexp_f32(1.0f, value_exponent);
            // The next step's loads go out before a step is computed (past the last step: of the last again). Two copies
            // of the body, so that each register of a step stays where it was loaded: a copy would wait for the loads.
            for (uint32_t n = 0; n < steps; n += 2) {
                load(st[1], min(n + 1, steps - 1));
                step(st[0], n);
                load(st[0], min(n + 2, steps - 1));
                if (n + 1 < steps) step(st[1], n + 1);
            }
            float bad = 0.0f;
#pragma unroll
            for (int j = 0; j < 2 * J; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) bad = fmaf(run.o[j][e], 0.0f, bad);
            if (!__any(bad != 0.0f)) break;  // 0 but where a sum is not finite
        }

        // the four lane groups hold different keys of one column
        float l = run.l, m = run.m;
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (l == 0.0f) m = kNone;
        if (g == 0) wave_ref[wave][c] = m;
        __syncthreads();
        // a row's reference: over the waves and its columns
        float ref = kNone;
#pragma unroll
        for (int k = 0; k < 4 * PACK; ++k) ref = fmaxf(ref, wave_ref[k / PACK][k % PACK * R + row]);
        const float f = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - ref);
        if (g == 0) wave_sum_l[wave][c] = l == 0.0f ? 0.0f : l * f;
        const float unscale = ldexp_f32(MODE == kFine ? 1.0f : 0x1p24f, -value_exponent);
        // lane: values 32 i + 8 g + 0 .. 7 of its column
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            float s = run.beta[gr];
            s += __shfl_xor(s, 16, 64);
            s += __shfl_xor(s, 32, 64);
#pragma unroll
            for (int i = gr * JG; i < (gr + 1) * JG; ++i) {
                float y[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float even = run.o[2 * i][e] - run.rounded[gr][e];
                    const float odd = fmaf(run.o[2 * i + 1][e], 0.0625f, -run.rounded[gr][e]);
                    y[2 * e] = l == 0.0f ? 0.0f : fmaf(even, unscale, s) * f;
                    y[2 * e + 1] = l == 0.0f ? 0.0f : fmaf(odd, unscale, s) * f;
                }
                // the two columns of a row: the 16-lane row rotated by 8
                if (PACK == 2) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] += dpp_f32<0x128>(y[e]);
                }
                if (pack == 0) {
                    float* dst = &sh.join[wave][row * kRow + 32 * i + 8 * g];
                    *(f32x4*)dst = f32x4{y[0], y[1], y[2], y[3]};
                    *(f32x4*)(dst + 4) = f32x4{y[4], y[5], y[6], y[7]};
                }
            }
        }
        __syncthreads();
        // the rows' values, N neighbouring ones to a thread
        constexpr int N = DIM * R / 256 < 4 ? 4 : DIM * R / 256;
        const uint32_t rr = threadIdx.x / (DIM / N), d = threadIdx.x % (DIM / N) * N;
        if (rr < R && row0 + rr < u.rows) {
            float v[N], sum = 0.0f;
#pragma unroll
            for (int e = 0; e < N; e += 4) {
                f32x4 s = *(const f32x4*)&sh.join[0][rr * kRow + d + e];
#pragma unroll
                for (int k = 1; k < 4; ++k) s += *(const f32x4*)&sh.join[k][rr * kRow + d + e];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[e + k] = s[k];
            }
            float rref = kNone;
#pragma unroll
            for (int k = 0; k < 4 * PACK; ++k) {
                sum += wave_sum_l[k / PACK][k % PACK * R + rr];
                rref = fmaxf(rref, wave_ref[k / PACK][k % PACK * R + rr]);
            }
            const uint32_t ti = (row0 + rr) * a.ratio_inverse >> 16, hh = head * a.ratio + row0 + rr - ti * a.ratio;
            const uint32_t tok = (uint32_t)u.r.first + ti;
            if (s0 == 0 && s1 == u.steps) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                uint16_t* p = (uint16_t*)a.out.p + (tok * a.out.token + hh * a.out.head + d);
#pragma unroll
                for (int e = 0; e < N; e += 4) store_out<4>(p + e, a.out.vec, a.is_bf16, v + e, inv);
                if (a.lse && d == 0)
                    a.lse[(size_t)tok * a.heads + hh] =
                        sum == 0.0f ? -INFINITY : (rref + __builtin_amdgcn_logf(sum)) * kLn2;
            } else {
                const size_t slot = (2 * (size_t)blockIdx.x + (s0 == 0)) * kRows + rr;
#pragma unroll
                for (int e = 0; e < N; e += 4) *(f32x4*)(a.po + slot * DIM + d + e) = f32x4{v[e], v[e + 1], v[e + 2], v[e + 3]};
                if (d == 0) a.pml[slot] = float2{rref, sum};
                if (s0 == 0 && threadIdx.x == 0)  // goes on in the workgroups up to the one that holds its last step
                    a.begun[blockIdx.x] = int4{u.r.first, (int)head, (int)(row0 | u.rows << 16), (int)((unit_end - 1) / per - blockIdx.x)};
            }
        }
        __syncthreads();  // the LDS buffers are free again
        if (threadIdx.x < 64) sh.q[J][threadIdx.x] = u32x4{0, 0, 0, 0};
    }
}

// A row of a unit that several workgroups share, by one wave: out = sum_w o_w 2^(m_w - m) / sum_w l_w 2^(m_w - m), in
// the order of the workgroups. Four rows a workgroup.
template <int DIM>
__global__ __launch_bounds__(256) void kv_attend_join(AttendArgs a) {
    constexpr int V = DIM / 64;  // values of a lane
    typedef float vec __attribute__((ext_vector_type(V)));
    const uint32_t quarters = a.row_block / 4, w = blockIdx.x / quarters, lane = threadIdx.x & 63;
    const uint32_t slot_row = blockIdx.x % quarters * 4 + (threadIdx.x >> 6);
    const int4 u = a.begun[w];
    if (u.x < 0) return;
    const uint32_t row = ((uint32_t)u.z & 0xffffu) + slot_row;
    if (row >= (uint32_t)u.z >> 16) return;
    const uint32_t i = row * a.ratio_inverse >> 16, token = (uint32_t)u.x + i, qh = (uint32_t)u.y * a.ratio + row - i * a.ratio;
    const uint32_t parts = (uint32_t)u.w + 1;
    // part 0 is the workgroup's last segment, part i the first of workgroup w + i
    const auto slot = [&](uint32_t i) { return (size_t)(i ? 2 * (w + i) : 2 * w + 1) * kRows + slot_row; };
    float m = kNone;
    for (uint32_t i = lane; i < parts; i += 64) m = fmaxf(m, a.pml[slot(i)].x);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    vec sum = 0.0f;
    float l = 0.0f;
#pragma unroll 8
    for (uint32_t i = 0; i < parts; ++i) {
        const float2 v = a.pml[slot(i)];
        const float f = __builtin_amdgcn_exp2f(v.x - m);
        l = fmaf(v.y, f, l);
        sum += *(const vec*)(a.po + slot(i) * DIM + V * lane) * f;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* p = (uint16_t*)a.out.p + (token * a.out.token + qh * a.out.head + V * lane);
#pragma unroll
    for (int e = 0; e < V; ++e)
        p[e] = a.is_bf16 ? f32_to_bf16_bits(sum[e] * inv) : f32_to_f16_bits(sum[e] * inv);
    if (a.lse && lane == 0) a.lse[(size_t)token * a.heads + qh] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

template <int DIM, int G, int PACK, int MODE>
stark_qmm_status launch(const AttendArgs& a, hipStream_t s) {
    const uint64_t units = (uint64_t)a.batch * a.cache.kv_heads * ((a.row_limit + a.row_block - 1) / a.row_block);
    hipLaunchKernelGGL((kv_attend_rows<DIM, G, PACK, MODE>), dim3(a.whole ? (uint32_t)units : a.grid), dim3(256), 0, s, a);
    QMM_HIP_CHECK(hipGetLastError());
    if (!a.whole) {
        hipLaunchKernelGGL((kv_attend_join<DIM>), dim3(a.grid * (a.row_block / 4)), dim3(256), 0, s, a);
        QMM_HIP_CHECK(hipGetLastError());
    }
    return STARK_QMM_OK;
}

template <int DIM, int G>
stark_qmm_status launch(const AttendArgs& a, hipStream_t s) {
    if (!a.is_bf16) return a.row_block == 8 ? launch<DIM, G, 2, kFine>(a, s) : launch<DIM, G, 1, kFine>(a, s);
    if (a.lse) return a.row_block == 8 ? launch<DIM, G, 2, kLse>(a, s) : launch<DIM, G, 1, kLse>(a, s);
    return a.row_block == 8 ? launch<DIM, G, 2, kPlain>(a, s) : launch<DIM, G, 1, kPlain>(a, s);
}

}  // namespace

namespace qmm {

stark_qmm_status launch_attend_rows(const AttendArgs& a, hipStream_t s) {
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
