// Attention over the 4-bit paged key/value cache (layout: kv_layout.h).
#include "kv_common.h"

namespace {

using namespace qmm;

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kNone = -1e30f;  // running maximum before any key

struct AttendArgs {
    KvCache cache;
    KvRows q, out;
    float* lse;
    const int32_t *table, *query_start, *kv_lengths;
    uint32_t batch, tokens, heads, ratio, stride, max_query, max_kv, tiles;
    float scale;    // of q . k: log2(e) * scale, or 2 log2(e) * scale / soft_cap
    float cap;      // soft_cap * log2(e), or 0
    uint32_t causal, window, is_bf16;
    uint32_t chunk, chunks;
    float* po;      // [token][head][chunk][dim] unnormalised partial outputs
    float2* pml;    // [token][head][chunk] (reference exponent, sum)
};

QMM_DEVICE float plane_scale(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[0]; }
QMM_DEVICE float plane_bias(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[1]; }

QMM_DEVICE f16x8 operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(f16x8, u32x4{a, b, c, d});
}

QMM_DEVICE kv::Request request_of(const AttendArgs& a, uint32_t b) {
    return kv::request(a.query_start[b], a.query_start[b + 1], a.kv_lengths[b], a.tokens, a.max_query, a.max_kv);
}

// N neighbouring output values, times f, at p; vec: 2 N bytes aligned.
template <int N>
QMM_DEVICE void store_out(uint16_t* p, uint32_t vec, uint32_t is_bf16, const float* x, float f) {
    uint32_t w[N / 2];
    if (is_bf16) {
#pragma unroll
        for (int e = 0; e < N / 2; ++e)
            w[e] = __builtin_bit_cast(uint32_t, bf16x2_t{(__bf16)(x[2 * e] * f), (__bf16)(x[2 * e + 1] * f)});
    } else {
#pragma unroll
        for (int e = 0; e < N / 2; ++e)
            w[e] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)(x[2 * e] * f), (_Float16)(x[2 * e + 1] * f)});
    }
    if (vec) {
        if (N == 8) *(u32x4*)p = u32x4{w[0], w[1], w[2 % (N / 2)], w[3 % (N / 2)]};
        else *(u32x2*)p = u32x2{w[0], w[1]};
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) p[e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
    }
}

// 32 keys of one kv head (two records) as a wave holds them: code words and plane words.
template <int DIM, int G>
struct Step {
    uint32_t kc[2][DIM / 32], vc[2][DIM / 32];
    u32x4 kp[2][G], vp[2][G];
    bool ok[2];  // the record's page is inside the cache

    // page: the two records' page ids; t0: first key
    QMM_DEVICE void load(const AttendArgs& a, const uint32_t (&page)[2], uint32_t head, uint32_t t0, uint32_t lane) {
        const uint32_t c = lane & 15, g = lane >> 4, mask = (1u << a.cache.page_shift) - 1;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            ok[i] = page[i] < a.cache.page_count;
            const uint8_t* rec = a.cache.data + kv::record_index(ok[i] ? page[i] : 0, a.cache.kv_heads, head, mask + 1,
                                                                  (t0 + 16 * i) & mask) * (uint64_t)a.cache.record;
            const uint8_t* kq = rec + (DIM == 64 ? c * 32 + g * 8 : c * 64 + g * 16);
            const uint8_t* vq = rec + 8 * DIM + 64 * G + lane * (DIM == 64 ? 8 : 16);
            if (DIM == 64) {
                *(u32x2*)&kc[i][0] = *(const u32x2*)kq;
                *(u32x2*)&vc[i][0] = *(const u32x2*)vq;
            } else {
#pragma unroll
                for (int h = 0; h < DIM / 128; ++h) {
                    *(u32x4*)&kc[i][4 * h] = *(const u32x4*)(kq + 1024 * h);
                    *(u32x4*)&vc[i][4 * h] = *(const u32x4*)(vq + 1024 * h);
                }
            }
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                kp[i][gr] = *(const u32x4*)(rec + 8 * DIM + 64 * gr + 16 * g);
                vp[i][gr] = *(const u32x4*)(rec + 16 * DIM + 64 * G + 64 * gr + 16 * g);
            }
        }
    }
};

// Page ids of a wave's records: lane 2 n + i holds that of record i of step base + n, 32 steps to a load, and a step
// reads its two with v_readlane.
struct PageIds {
    const int32_t* row;
    int32_t from, stride;  // first key of step 0; keys from a wave's step to its next
    uint32_t shift, last;  // last entry of the table row
    uint32_t ids, base;

    QMM_DEVICE void fill(uint32_t n, uint32_t lane) {
        base = n;
        const uint32_t t = (uint32_t)(from + stride * (int32_t)(n + lane / 2)) + 16 * (lane & 1);
        ids = (uint32_t)row[min(t >> shift, last)];  // a step may reach past the last key: past the table too
        asm volatile("" : "+v"(ids));  // the wait for it is here, not before every v_readlane (for all loads in flight)
    }
    QMM_DEVICE void get(uint32_t n, uint32_t lane, uint32_t (&page)[2]) {
        if (n - base >= 32) fill(n, lane);
        page[0] = (uint32_t)__builtin_amdgcn_readlane((int)ids, (int)(2 * (n - base)));
        page[1] = (uint32_t)__builtin_amdgcn_readlane((int)ids, (int)(2 * (n - base) + 1));
    }
};

// Running state of 16 query rows: lane (c, g) holds row c.
template <int DIM, int G>
struct Running {
    static constexpr int J = DIM / 32, JG = J / G;
    f32x4 o[2 * J];          // [32-value block, parity]: codes times p s, values 32 i + 2 (4 g + e) + parity
    float beta[G], l, m, mf; // sum p b and sum p over the lane's keys; reference; reference - exponent
    int fexp;

    QMM_DEVICE void start(int exponent) {
        fexp = exponent;
        m = kNone, mf = kNone - (float)exponent, l = 0.0f;
#pragma unroll
        for (int j = 0; j < 2 * J; ++j) o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int gr = 0; gr < G; ++gr) beta[gr] = 0.0f;
    }
};

// Rows of a tile by 32-key steps, the steps dealt to four waves, each with its own running maximum and sums, joined
// at the end. Keys and values stay codes: with C the codes,
//   q . k = sum over groups (s_g C_g . q + b_g sum q),   out = sum over tokens (p s_g) C + sum p b_g,
// so a key's scale and bias are two fma per score and group, a value's scale goes into the probability (f16, p s_g
// scaled by a power of two that keeps it in f16's normal range), and a code becomes an f16 operand by a mask: the bits
// of c in the low (or 4 bits higher) end of an f16 are the subnormal c 2^-24 (c 2^-20), exact.
// Scores come out transposed (A rows = keys, B columns = query rows): a lane holds four keys of one query row in each
// record, which is the B operand of the second product as it stands, with no lane exchange.
// q is scaled per row by a power of two into f16's range, exact but for values 2^-24 below the row's largest.
template <int DIM, int G>
__global__ __launch_bounds__(256, DIM == 256 ? 1 : 2) void kv_attend_rows(AttendArgs a) {
    constexpr int J = DIM / 32;       // k blocks of a score product, and 32-value blocks of the output
    constexpr int JG = J / G;         // of one scale group
    constexpr int kRow = DIM + 4;     // padded row of the joining buffers, floats
    __shared__ float join[2][16 * kRow];
    __shared__ float wave_ref[4][16], wave_sum_l[4][16];
    const uint32_t lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t id = blockIdx.x;
    const uint32_t tile = id % a.tiles;
    id /= a.tiles;
    const uint32_t head = id % a.cache.kv_heads;
    id /= a.cache.kv_heads;
    const uint32_t b = id % a.batch, part = id / a.batch;
    const kv::Request r = request_of(a, b);
    const uint32_t rows = (uint32_t)r.q_len * a.ratio;
    if (tile * kv::kRows >= rows) return;
    const kv::Range span = kv::tile_range(tile, a.ratio, r.q_len, r.kv_len, a.causal, a.window);
    const uint64_t cut0 = (uint64_t)part * a.chunk, cut1 = cut0 + a.chunk;
    const int32_t from = max(span.lo & ~31, (int32_t)min(cut0, (uint64_t)0x7fffffff));
    const int32_t to = (int32_t)min((uint64_t)span.hi, cut1);
    if (from >= to && a.chunks > 1) return;  // the join skips it too

    const uint32_t rho = tile * kv::kRows + c;
    const bool live = rho < rows;
    const uint32_t qi = live ? rho / a.ratio : 0, qh = head * a.ratio + (live ? rho % a.ratio : 0);
    const uint32_t token = (uint32_t)r.first + qi;
    kv::Range see = kv::visible((int32_t)qi, r.q_len, r.kv_len, a.causal, a.window);
    if (!live) see = {0, 0x7fffffff};

    // B operands of the score products: lane group g holds dims 8 (4 j + g) .. + 7, in the order of the code pairs
    f16x8 qb[J];
    float qsum[G];
    float c1;
    {
        // a row past the tile's last reads the request's first one, as zeros
        u32x4 w[J];
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
        float x[J][8];
        if (a.is_bf16) {
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    x[j][e] = __uint_as_float(e & 1 ? w[j][e / 2] & 0xffff0000u : w[j][e / 2] << 16);
        } else {
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[j][e] = (float)__builtin_bit_cast(f16x2, (uint32_t)w[j][e / 2])[e & 1];
        }
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[j][e] = live ? x[j][e] : 0.0f;
                top = fmaxf(top, fabsf(x[j][e]));
            }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const int k = 13 - (top > 0.0f && top < INFINITY ? ilogbf(top) : 0);  // the largest in [2^13, 2^14)
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            float s = 0.0f;
#pragma unroll
            for (int j = gr * JG; j < (gr + 1) * JG; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) s += x[j][e];
            s += __shfl_xor(s, 16, 64);
            s += __shfl_xor(s, 32, 64);
            qsum[gr] = s * a.scale;
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            // code pairs of a word: nibbles (0, 4), (1, 5) sixteenfold, (2, 6), (3, 7) sixteenfold
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int n = e / 2 + 4 * (e & 1);
                qb[j][e] = (_Float16)ldexp_f32(x[j][n], (e / 2) & 1 ? k - 4 : k);
            }
        }
        c1 = ldexp_f32(a.scale, 24 - k);
    }

    // this wave's 32-key steps: wave, wave + 4, ...
    const int32_t all_steps = from < to ? (to - from + 31) / 32 : 0;
    const uint32_t steps = (int32_t)wave < all_steps ? (uint32_t)(all_steps - (int32_t)wave + 3) / 4 : 0;
    // keys that every row of the tile sees: [inner_lo, inner_hi)
    const kv::Range first = kv::visible((int32_t)(tile * kv::kRows / a.ratio), r.q_len, r.kv_len, a.causal, a.window);
    const kv::Range last = kv::visible((int32_t)(min(tile * kv::kRows + kv::kRows, rows) - 1) / (int32_t)a.ratio,
                                       r.q_len, r.kv_len, a.causal, a.window);
    const int32_t inner_lo = last.lo, inner_hi = min(first.hi, last.hi);
    PageIds pages{a.table + (size_t)b * a.stride, from + 32 * (int32_t)wave, 128, a.cache.page_shift, a.stride - 1, 0, 0};

    Running<DIM, G> run;
    run.start(0);

    const auto load = [&](Step<DIM, G>& st, uint32_t n) {
        uint32_t page[2];
        pages.get(n, lane, page);
        st.load(a, page, head, (uint32_t)(from + 32 * (int32_t)wave + 128 * (int32_t)n), lane);
    };
    // largest value scale (f16 bits) of the step's keys before `to`
    const auto scale_max = [&](const Step<DIM, G>& st, uint32_t n, uint32_t smax) {
        const int32_t t0 = from + 32 * (int32_t)wave + 128 * (int32_t)n;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int gr = 0; gr < G; ++gr)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t h = st.vp[i][gr][e] & 0xffffu;
                    if (t0 + 16 * i + 4 * (int32_t)g + e < to && h < 0x7c00u && st.ok[i]) smax = max(smax, h);
                }
        return smax;
    };
    const auto exponent = [&](uint32_t smax) {
        smax = group_max<16>(smax);
        smax = max(smax, (uint32_t)__shfl_xor((int)smax, 16, 64));
        smax = max(smax, (uint32_t)__shfl_xor((int)smax, 32, 64));
        return smax ? 8 - ilogbf(f16_bits_to_f32(smax)) : 0;
    };
    const auto step = [&](Step<DIM, G>& st, uint32_t n) {
        const int32_t t0 = from + 32 * (int32_t)wave + 128 * (int32_t)n;
        float x[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f32x4 acc[G];
#pragma unroll
            for (int gr = 0; gr < G; ++gr) acc[gr] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const uint32_t w = st.kc[i][j], v = w >> 8;
                const f16x8 k = operand(w & 0x000f000fu, w & 0x00f000f0u, v & 0x000f000fu, v & 0x00f000f0u);
                acc[j / JG] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qb[j], acc[j / JG], 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float y = 0.0f, z = 0.0f;
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    y = fmaf(plane_scale(st.kp[i][gr][e]), acc[gr][e], y);
                    z = fmaf(plane_bias(st.kp[i][gr][e]), qsum[gr], z);
                }
                x[i][e] = fmaf(y, c1, z);
            }
        }
        if (a.cap != 0.0f) {  // cap tanh(s / cap) = cap (1 - 2 / (1 + e^(2 s / cap)))
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    x[i][e] = a.cap - 2.0f * a.cap * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x[i][e]));
        }
        if (t0 < inner_lo || t0 + 32 > inner_hi || !st.ok[0] || !st.ok[1]) {
            // keys that a row does not see: score -inf, and planes 0, so that nothing of theirs (a NaN) gets through
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int32_t t = t0 + 16 * i + 4 * (int32_t)g + e;
                    const bool seen = t >= see.lo && t < see.hi && t < to && st.ok[i];
                    x[i][e] = seen ? x[i][e] : -INFINITY;
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) st.vp[i][gr][e] = seen ? st.vp[i][gr][e] : 0u;
                }
        }
        float top = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])),
                          fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
        // the reference moves only when a score passes it by 2^6: rescaling is then rare
        if (__any(top > run.m + 6.0f)) {
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float mn = fmaxf(run.m, top), f = __builtin_amdgcn_exp2f(run.m - mn);
            run.m = mn;
            run.mf = mn - (float)run.fexp;
            run.l *= f;
#pragma unroll
            for (int gr = 0; gr < G; ++gr) run.beta[gr] *= f;
#pragma unroll
            for (int j = 0; j < 2 * J; ++j) run.o[j] *= f;
        }
        f16x8 ps[G];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p = __builtin_amdgcn_exp2f(x[i][e] - run.mf);
                run.l += p;
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    // p s to f16, half a unit of 2^-11: the codes it multiplies are exact
                    ps[gr][4 * i + e] = (_Float16)(p * plane_scale(st.vp[i][gr][e]));
                    run.beta[gr] = fmaf(p, plane_bias(st.vp[i][gr][e]), run.beta[gr]);
                }
            }
#pragma unroll
        for (int i = 0; i < J; ++i) {  // 32-value blocks; byte i of a lane's value words
            uint32_t w[4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (DIM == 64) {
                    const uint32_t sel = 0x0c000c00u | (uint32_t)(2 + i) << 16 | (uint32_t)i;
                    w[2 * u] = permb(0, st.vc[u][0], sel);
                    w[2 * u + 1] = permb(0, st.vc[u][1], sel);
                } else {
                    const uint32_t sel = 0x0c000c00u | (uint32_t)(4 + i % 4) << 16 | (uint32_t)(i % 4);
                    const uint32_t* v = &st.vc[u][i / 4 * 4];
                    w[2 * u] = permb(v[1], v[0], sel);
                    w[2 * u + 1] = permb(v[3], v[2], sel);
                }
            }
            const f16x8 lo = operand(w[0] & 0x000f000fu, w[1] & 0x000f000fu, w[2] & 0x000f000fu, w[3] & 0x000f000fu);
            const f16x8 hi = operand(w[0] & 0x00f000f0u, w[1] & 0x00f000f0u, w[2] & 0x00f000f0u, w[3] & 0x00f000f0u);
            run.o[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, ps[i / JG], run.o[2 * i], 0, 0, 0);
            run.o[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, ps[i / JG], run.o[2 * i + 1], 0, 0, 0);
        }
    };

    // Power of two on the probabilities: p s below 2^15 while p < 2^6, taken from the scales of the wave's first step.
    // Should a later scale be far larger, the products overflow to infinity, which shows in the sums at the end:
    // then the wave starts again with the largest scale of all its steps.
    for (int attempt = 0; attempt < 2 && steps; ++attempt) {
        Step<DIM, G> st[2];
        uint32_t smax = 0;
        if (attempt) {
            for (uint32_t n = 0; n < steps; ++n) {
                load(st[0], n);
                smax = scale_max(st[0], n, smax);
            }
        }
        // the next step's loads go out before a step is computed (past the last step: the last again)
        pages.fill(0, lane);
        load(st[0], 0);
        if (!attempt) smax = scale_max(st[0], 0, 0);
        run.start(exponent(smax));
        for (uint32_t n = 0; n < steps; n += 2) {
            load(st[1], min(n + 1, steps - 1));
            step(st[0], n);
            if (n + 1 >= steps) break;
            load(st[0], min(n + 2, steps - 1));
            step(st[1], n + 1);
        }
        float bad = 0.0f;
#pragma unroll
        for (int j = 0; j < 2 * J; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) bad = fmaf(run.o[j][e], 0.0f, bad);
        if (!__any(bad != 0.0f)) break;  // 0 but where a sum is not finite
    }
    float l = run.l, mf = run.mf;
    auto& o = run.o;
    auto& beta = run.beta;

    // the four lane groups hold different keys of one row
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
        beta[gr] += __shfl_xor(beta[gr], 16, 64);
        beta[gr] += __shfl_xor(beta[gr], 32, 64);
    }
    if (l == 0.0f) mf = kNone;
    if (g == 0) wave_ref[wave][c] = mf;
    __syncthreads();
    const float ref = fmaxf(fmaxf(wave_ref[0][c], wave_ref[1][c]), fmaxf(wave_ref[2][c], wave_ref[3][c]));
    const float f = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(mf - ref);
    if (g == 0) wave_sum_l[wave][c] = l == 0.0f ? 0.0f : l * f;
    // lane: values 32 i + 8 g + 0 .. 7 of row c
    float y[J][8];
#pragma unroll
    for (int i = 0; i < J; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            y[i][2 * e] = l == 0.0f ? 0.0f : fmaf(o[2 * i][e], 0x1p24f, beta[i / JG]) * f;
            y[i][2 * e + 1] = l == 0.0f ? 0.0f : fmaf(o[2 * i + 1][e], 0x1p20f, beta[i / JG]) * f;
        }
#pragma unroll
    for (int half = 2; half >= 1; half >>= 1) {  // waves 2, 3 to 0, 1; then 1 to 0
        if ((int)wave >= half && (int)wave < 2 * half) {
            float* dst = &join[wave - half][c * kRow + 8 * g];
#pragma unroll
            for (int i = 0; i < J; ++i) {
                *(f32x4*)(dst + 32 * i) = f32x4{y[i][0], y[i][1], y[i][2], y[i][3]};
                *(f32x4*)(dst + 32 * i + 4) = f32x4{y[i][4], y[i][5], y[i][6], y[i][7]};
            }
        }
        __syncthreads();
        if ((int)wave < half) {
            const float* src = &join[wave][c * kRow + 8 * g];
#pragma unroll
            for (int i = 0; i < J; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) y[i][e] += src[32 * i + e];
        }
        __syncthreads();
    }
    if (wave != 0 || !live) return;
    const float sum = (wave_sum_l[0][c] + wave_sum_l[1][c]) + (wave_sum_l[2][c] + wave_sum_l[3][c]);
    if (a.chunks == 1) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        uint16_t* p = (uint16_t*)a.out.p + (token * a.out.token + qh * a.out.head + 8 * g);
#pragma unroll
        for (int i = 0; i < J; ++i) store_out<8>(p + 32 * i, a.out.vec, a.is_bf16, y[i], inv);
        if (a.lse && g == 0)
            a.lse[(size_t)token * a.heads + qh] = sum == 0.0f ? -INFINITY : (ref + __builtin_amdgcn_logf(sum)) * kLn2;
    } else {
        const size_t at = ((size_t)token * a.heads + qh) * a.chunks + part;
        float* dst = a.po + at * DIM + 8 * g;
#pragma unroll
        for (int i = 0; i < J; ++i) {
            *(f32x4*)(dst + 32 * i) = f32x4{y[i][0], y[i][1], y[i][2], y[i][3]};
            *(f32x4*)(dst + 32 * i + 4) = f32x4{y[i][4], y[i][5], y[i][6], y[i][7]};
        }
        if (g == 0) a.pml[at] = float2{ref, sum};
    }
}

// The chunks of one row: out = sum_c o_c 2^(m_c - m) / sum_c l_c 2^(m_c - m). 256 threads: DIM / 4 columns of four
// values, the chunks dealt to the rest and added in a fixed order.
template <int DIM>
__global__ __launch_bounds__(256) void kv_attend_join(AttendArgs a) {
    constexpr uint32_t COLS = DIM / 4, SUBS = 256 / COLS;
    __shared__ f32x4 acc[SUBS][COLS];
    __shared__ float red[2][4];
    uint32_t id = blockIdx.x;
    const uint32_t qh = id % a.heads;
    id /= a.heads;
    const uint32_t qi = id % a.max_query, b = id / a.max_query;
    const kv::Request r = request_of(a, b);
    if ((int32_t)qi >= r.q_len) return;
    const uint32_t token = (uint32_t)r.first + qi;
    const kv::Range span = kv::tile_range((qi * a.ratio + qh % a.ratio) / kv::kRows, a.ratio, r.q_len, r.kv_len,
                                          a.causal, a.window);
    // the chunks that hold a key of the row's tile: exactly those the tile's workgroups wrote
    const uint32_t c0 = (uint32_t)span.lo / a.chunk, c1 = span.hi > span.lo ? ((uint32_t)span.hi + a.chunk - 1) / a.chunk : c0;
    const size_t base = ((size_t)token * a.heads + qh) * a.chunks;
    const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6;
    float m = kNone;
    for (uint32_t c = c0 + t; c < c1; c += 256) m = fmaxf(m, a.pml[base + c].x);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    if (lane == 0) red[0][wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    float l = 0.0f;
    for (uint32_t c = c0 + t; c < c1; c += 256) {
        const float2 v = a.pml[base + c];
        l += v.y * __builtin_amdgcn_exp2f(v.x - m);
    }
    l = wave_sum(l);
    if (lane == 0) red[1][wave] = l;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t col = t % COLS, sub = t / COLS;
    for (uint32_t c = c0 + sub; c < c1; c += SUBS) {
        const float f = __builtin_amdgcn_exp2f(a.pml[base + c].x - m);
        sum += *(const f32x4*)(a.po + (base + c) * DIM + 4 * col) * f;
    }
    acc[sub][col] = sum;
    __syncthreads();
    l = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    if (sub == 0) {
        for (uint32_t s = 1; s < SUBS; ++s) sum += acc[s][col];
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint16_t* p = (uint16_t*)a.out.p + (token * a.out.token + qh * a.out.head + 4 * col);
        const float y[4] = {sum[0], sum[1], sum[2], sum[3]};
        store_out<4>(p, a.out.vec, a.is_bf16, y, inv);
        if (a.lse && col == 0)
            a.lse[(size_t)token * a.heads + qh] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
    }
}

template <int DIM, int G>
stark_qmm_status launch_rows(const AttendArgs& a, hipStream_t s) {
    const uint64_t blocks = (uint64_t)a.tiles * a.cache.kv_heads * a.batch * a.chunks;
    if (blocks >= 1ull << 24) return STARK_QMM_UNSUPPORTED;
    hipLaunchKernelGGL((kv_attend_rows<DIM, G>), dim3((uint32_t)blocks), dim3(256), 0, s, a);
    QMM_HIP_CHECK(hipGetLastError());
    if (a.chunks > 1) {
        const uint64_t joins = (uint64_t)a.heads * a.max_query * a.batch;
        if (joins >= 1ull << 24) return STARK_QMM_UNSUPPORTED;
        hipLaunchKernelGGL((kv_attend_join<DIM>), dim3((uint32_t)joins), dim3(256), 0, s, a);
        QMM_HIP_CHECK(hipGetLastError());
    }
    return STARK_QMM_OK;
}

// Checks all but the pointers, which a size query need not have; fills the lengths.
stark_qmm_status check(const stark_qmm_kv_attention_args* p, AttendArgs* a) {
    if (!p) return STARK_QMM_INVALID_ARGUMENT;
    if (p->struct_size != sizeof(*p)) return STARK_QMM_ABI_MISMATCH;
    uint64_t bytes;
    const stark_qmm_status st = kv_geometry(p->cache, &a->cache, &bytes);
    if (st != STARK_QMM_OK) return st;
    if (p->data_type != STARK_QMM_F16 && p->data_type != STARK_QMM_BF16) return STARK_QMM_UNSUPPORTED_DATA_TYPE;
    if (p->heads == 0 || p->heads > 65536 || p->heads % a->cache.kv_heads) return STARK_QMM_INVALID_ARGUMENT;
    if (p->batch > (1u << 20) || p->tokens > (1u << 24) || p->max_kv > 0x7fffffffu) return STARK_QMM_INVALID_ARGUMENT;
    if ((uint64_t)p->table_stride * p->cache.page_size > 0x7fffffffull || p->table_stride == 0)
        return STARK_QMM_INVALID_ARGUMENT;
    if (!(p->soft_cap >= 0.0f) || !(p->soft_cap < INFINITY) || !(fabsf(p->scale) < INFINITY))
        return STARK_QMM_INVALID_ARGUMENT;
    a->batch = p->batch, a->tokens = p->tokens, a->heads = p->heads, a->ratio = p->heads / a->cache.kv_heads;
    a->stride = p->table_stride;
    a->max_query = std::min(p->max_query, p->tokens);
    a->max_kv = std::min(p->max_kv, p->table_stride * p->cache.page_size);
    a->tiles = (uint32_t)(((uint64_t)a->max_query * a->ratio + kv::kRows - 1) / kv::kRows);
    a->is_bf16 = p->data_type == STARK_QMM_BF16;
    a->causal = p->causal != 0, a->window = p->window;
    a->scale = p->soft_cap != 0.0f ? 2.0f * kLog2e * p->scale / p->soft_cap : kLog2e * p->scale;
    a->cap = p->soft_cap * kLog2e;
    return STARK_QMM_OK;
}

// The split of the checked call, and the bytes that its partial results need.
stark_qmm_status plan_split(AttendArgs* a, uint64_t* workspace) {
    int dev = 0, cus = 0;
    QMM_HIP_CHECK(hipGetDevice(&dev));
    QMM_HIP_CHECK(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
    const uint64_t units = std::max<uint64_t>(1, (uint64_t)a->batch * a->cache.kv_heads * a->tiles);
    const kv::Split s = kv::split(units, a->max_kv, (uint32_t)cus);
    a->chunk = s.chunk, a->chunks = s.chunks;
    *workspace = s.chunks > 1 ? (uint64_t)a->tokens * a->heads * s.chunks * (a->cache.dim * 4ull + 8) : 0;
    return STARK_QMM_OK;
}

}  // namespace

extern "C" {

stark_qmm_status stark_qmm_kv_attention_workspace_size(const stark_qmm_kv_attention_args* args, uint64_t* bytes) {
    AttendArgs a{};
    if (!bytes) return STARK_QMM_INVALID_ARGUMENT;
    const stark_qmm_status st = check(args, &a);
    return st != STARK_QMM_OK ? st : plan_split(&a, bytes);
}

stark_qmm_status stark_qmm_kv_attention(const stark_qmm_kv_attention_args* p, void* stream) {
    AttendArgs a{};
    stark_qmm_status st = check(p, &a);
    if (st != STARK_QMM_OK) return st;
    st = kv_view(p->cache, &a.cache);
    if (st != STARK_QMM_OK) return st;
    if (a.batch == 0 || a.max_query == 0) return STARK_QMM_OK;
    if (!p->query_start || !p->kv_lengths || !p->block_table || !kv_aligned(p->query_start, 4) ||
        !kv_aligned(p->kv_lengths, 4) || !kv_aligned(p->block_table, 4) || !kv_aligned(p->lse, 4))
        return STARK_QMM_INVALID_ARGUMENT;
    if (!kv_rows_ok(p->q, p->q_token_stride, p->q_head_stride, a.tokens, a.heads, a.cache.dim, p->data_type) ||
        !kv_rows_ok(p->out, p->out_token_stride, p->out_head_stride, a.tokens, a.heads, a.cache.dim, p->data_type))
        return STARK_QMM_INVALID_ARGUMENT;
    uint64_t need = 0;
    st = plan_split(&a, &need);
    if (st != STARK_QMM_OK) return st;
    if (need && (!p->workspace || !kv_aligned(p->workspace, 16))) return STARK_QMM_INVALID_ARGUMENT;
    if (need > p->workspace_size) return STARK_QMM_WORKSPACE_TOO_SMALL;
    a.q = kv_rows(p->q, p->q_token_stride, p->q_head_stride, p->data_type);
    a.out = kv_rows(p->out, p->out_token_stride, p->out_head_stride, p->data_type);
    a.lse = p->lse;
    a.table = p->block_table, a.query_start = p->query_start, a.kv_lengths = p->kv_lengths;
    if (need) {
        a.po = (float*)p->workspace;
        a.pml = (float2*)(a.po + (uint64_t)a.tokens * a.heads * a.chunks * a.cache.dim);
    }
    const hipStream_t s = (hipStream_t)stream;
    switch (a.cache.dim * 16 + a.cache.groups) {
    case 64 * 16 + 1: return launch_rows<64, 1>(a, s);
    case 64 * 16 + 2: return launch_rows<64, 2>(a, s);
    case 128 * 16 + 1: return launch_rows<128, 1>(a, s);
    case 128 * 16 + 2: return launch_rows<128, 2>(a, s);
    case 128 * 16 + 4: return launch_rows<128, 4>(a, s);
    case 256 * 16 + 2: return launch_rows<256, 2>(a, s);
    case 256 * 16 + 4: return launch_rows<256, 4>(a, s);
    default: return launch_rows<256, 8>(a, s);
    }
}

}  // extern "C"
