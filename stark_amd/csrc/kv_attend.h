// Shared by the attention kernels over the 4-bit paged key/value cache.
#pragma once

#include <float.h>

#include "kv_common.h"

namespace qmm {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kNone = -FLT_MAX;  // running maximum before any key: no score is below it
constexpr uint32_t kRows = 16;   // query rows of a matrix-core column block

struct AttendArgs {
    KvCache cache;
    KvRows q, out;
    float* lse;
    const int32_t *table, *query_start, *kv_lengths;
    uint32_t batch, tokens, heads, ratio, stride, max_query, max_kv;
    float scale;    // of q . k: log2(e) * |scale|, or 2 log2(e) * |scale| / soft_cap; 1 for a scale of 0
    float sign;     // of the scale: 1, -1 or 0; it goes to q
    float cap;      // soft_cap * log2(e), or 0
    uint32_t causal, is_bf16;
    int32_t window;
    // decode rows (kv_attend_rows)
    uint32_t row_limit;      // requests with more rows to a kv head are kv_attend_tiles's; 0: all are
    uint32_t row_block;      // 8 or 16
    uint32_t ratio_inverse;  // ceil(65536 / ratio): x / ratio for x < 64 and ratios up to 64
    uint32_t whole;          // a unit to a workgroup, no partial results
    uint32_t grid, inverse;  // else the workgroups that share the steps, and 2^32 / grid
    float* po;               // [2 grid][16 rows][dim] unnormalised partial outputs
    float2* pml;             // [2 grid][16 rows] (reference exponent, sum)
    int4* begun;             // [grid] unit that begins in a workgroup and goes on in later ones: its request's first token
                             // (-1: none), head, first row | rows of the request << 16, later ones
    // rows of prompts (kv_attend_tiles)
    uint32_t tiles;             // workgroups of a request, where that is no more than turns; else 0
    uint32_t turns;             // workgroups of a kv head (and piece)
    uint32_t pieces;            // that a tile's keys may be cut into
    float* tile_po;             // [token][head][piece][dim] unnormalised partial outputs
    float2* tile_pml;           // [token][head][piece] (reference exponent, sum)
};

QMM_DEVICE float plane_scale(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[0]; }
QMM_DEVICE float plane_bias(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[1]; }
// bias + 8 scale: the value of code 8
QMM_DEVICE float plane_middle(uint32_t w) { return fmaf(plane_scale(w), 8.0f, plane_bias(w)); }

// Soft cap of scores: cap tanh(u), u = x ln(2) / 2, of x = 2 log2(e) s / soft_cap, with cap = soft_cap log2(e).
// 1 - 2 / (1 + e^(2 u)) is off by some 2^-23 beside 1 for any u: a score by 2^-22 of the cap. Caps up to 64 take it as it is
// (1.5e-5, less than the f32 sums of a score may leave); a larger cap would swallow small scores, so there u below 0.3 takes
// the power series of tanh up to u^9, off by 2^-24 of itself, and a score is right to 2^-20 of itself. (The series for every
// cap: 52.5 us instead of 43.8 for 12 requests of 1 to 701 tokens under a cap of 30.)
constexpr float kPlainCap = 64.0f * kLog2e;
QMM_DEVICE float soft_capped(float x, float cap) {
    return fmaf(-2.0f * cap, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x)), cap);
}
QMM_DEVICE float soft_capped_exact(float x, float cap) {
    constexpr float h = 0.5f * kLn2, h2 = h * h;
    const float w = x * x;
    const float p = fmaf(w, fmaf(w, fmaf(w, 62.0f / 2835.0f * h2 * h2 * h2 * h2, -17.0f / 315.0f * h2 * h2 * h2), 2.0f / 15.0f * h2 * h2),
                         -1.0f / 3.0f * h2);
    return w < 0.75f ? cap * h * x * fmaf(w, p, 1.0f) : soft_capped(x, cap);
}

QMM_DEVICE f16x8 operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(f16x8, u32x4{a, b, c, d});
}

QMM_DEVICE kv::Request request_of(const AttendArgs& a, uint32_t b) {
    return kv::request(a.query_start[b], a.query_start[b + 1], a.kv_lengths[b], a.tokens, a.max_query, a.max_kv);
}

// N pieces of eight values of a q row as f32.
template <int N>
QMM_DEVICE void widen(const u32x4 (&w)[N], uint32_t is_bf16, float (&x)[N][8]) {
    if (is_bf16) {
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[j][e] = __uint_as_float(e & 1 ? w[j][e / 2] & 0xffff0000u : w[j][e / 2] << 16);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[j][e] = (float)__builtin_bit_cast(f16x2, (uint32_t)w[j][e / 2])[e & 1];
    }
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

// Launchers (kv_attend_rows.hip, kv_attend_tiles.hip).
stark_qmm_status launch_attend_rows(const AttendArgs& a, hipStream_t stream);
stark_qmm_status launch_attend_tiles(const AttendArgs& a, hipStream_t stream);

}  // namespace qmm
