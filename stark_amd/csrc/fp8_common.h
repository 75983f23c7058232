// Shared by the products of 8-bit floating-point codes (fp8_*.hip).
#pragma once

#include "qmm_common.h"

#include "fp8_layout.h"

namespace qmm {

// A checked product: `experts` groups of rows (one group of all rows where group_start is null).
struct Fp8Product {
    const uint8_t* a;
    const uint8_t* b;
    const float* as;
    const float* bs;
    void* d;
    const void* bias;
    const int32_t* group_start;
    const int32_t* a_rows;
    uint64_t a_stride, b_stride, b_expert;                         // bytes
    uint64_t as_row, as_block, bs_row, bs_block, bs_expert;        // elements
    uint64_t d_stride, bias_expert;                                // elements
    uint32_t m, n, k, experts, a_row_count;
    uint32_t d_dt, flags;
    float ab_scale, soft_cap;
    uint32_t vec;  // four outputs of a row may be stored at once
};

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Bytes of two row ranges [rows, width] (width and stride in bytes) meet.
inline bool fp8_overlap(const void* p, uint64_t pn, const void* q, uint64_t qn) {
    return p && q && pn && qn && (uintptr_t)p < (uintptr_t)q + qn && (uintptr_t)q < (uintptr_t)p + pn;
}
inline uint64_t fp8_span(uint64_t rows, uint64_t stride, uint64_t width) { return rows ? (rows - 1) * stride + width : 0; }
inline bool fp8_aligned(const void* p, uint64_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
inline uint64_t fp8_element(uint32_t dt) { return dt == STARK_QMM_F32 ? 4 : 2; }
inline bool fp8_type(uint32_t dt) { return dt == STARK_QMM_F32 || dt == STARK_QMM_F16 || dt == STARK_QMM_BF16; }

// A 16 x 16 block of A B over 128 codes, from zero: lane l has row (column) l % 16 of A (B) and 32 of its codes (which 32 does
// not matter while both operands agree), and outputs (4 (l / 16) + e, l % 16).
//
// v_mfma_f32_16x16x128_f8f6f4 takes codes as they are. It adds products in groups of eight neighbouring codes, and what a
// product has below 2^-13 of the largest product's binade in its group is cut off before the sum (measured; sums of groups are
// f32): outputs of normally distributed codes are off by 1.5e-5 of their size, which one of 8 or 11 bits does not show
// (1.7e-3 and 2e-4 by its own rounding). f32 outputs would: their codes are widened to bf16 first, exactly, and
// v_mfma_f32_16x16x32_bf16 adds in f32 (1e-8), at half the rate.
typedef __bf16 fp8_bf16x8 __attribute__((ext_vector_type(8)));
template <bool EXACT>
struct Fp8Operand {
    i32x8 v;
    QMM_DEVICE Fp8Operand() {}
    QMM_DEVICE explicit Fp8Operand(i32x8 x) : v(x) {}
};
template <>
struct Fp8Operand<true> {
    fp8_bf16x8 v[4];
    QMM_DEVICE Fp8Operand() {}
    QMM_DEVICE explicit Fp8Operand(i32x8 x) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const auto lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)x[i], 1.0f, false);
            const auto hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)x[i], 1.0f, true);
            v[i / 2][4 * (i % 2)] = lo[0], v[i / 2][4 * (i % 2) + 1] = lo[1];
            v[i / 2][4 * (i % 2) + 2] = hi[0], v[i / 2][4 * (i % 2) + 3] = hi[1];
        }
    }
};
QMM_DEVICE f32x4 fp8_block(const Fp8Operand<false>& a, const Fp8Operand<false>& b) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, f32x4{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
}
QMM_DEVICE f32x4 fp8_block(const Fp8Operand<true>& a, const Fp8Operand<true>& b) {
    f32x4 c = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
}

// One output as stark_qmm_encode finishes it.
QMM_DEVICE float fp8_finish(const Fp8Product& p, float sum, size_t d_at, const void* bias, uint32_t n) {
    float v = p.ab_scale * sum;
    if (p.flags & FLAG_ACCUMULATE) v += load_as_f32(p.d, p.d_dt, d_at);
    if (bias) v += load_as_f32(bias, p.d_dt, n);
    if (p.flags & FLAG_SOFT_CAP) v = p.soft_cap * tanhf(v / p.soft_cap);
    return v;
}

// Four consecutive outputs of a row from column n on.
QMM_DEVICE void fp8_store4(const Fp8Product& p, f32x4 sum, uint32_t row, uint32_t n, const void* bias) {
    const size_t at = (size_t)row * p.d_stride + n;
    if (n >= p.n) return;
    if (!p.vec || n + 4 > p.n) {
#pragma unroll 1
        for (uint32_t e = 0; e < 4 && n + e < p.n; ++e) {
            const float x = e == 0 ? sum[0] : e == 1 ? sum[1] : e == 2 ? sum[2] : sum[3];
            store_from_f32(p.d, p.d_dt, at + e, fp8_finish(p, x, at + e, bias, n + e));
        }
        return;
    }
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = p.ab_scale * sum[e];
    if (p.flags || bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fp8_finish(p, sum[e], at + e, bias, n + e);
    }
    if (p.d_dt == STARK_QMM_F32) {
        *(f32x4*)((float*)p.d + at) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
        uint32_t h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = p.d_dt == STARK_QMM_BF16 ? f32_to_bf16_bits(v[e]) : f32_to_f16_bits(v[e]);
        *(uint2*)((uint16_t*)p.d + at) = uint2{h[0] | (h[1] << 16), h[2] | (h[3] << 16)};
    }
}

// The rows of one row tile: expert, first row of d, rows (0: no tile).
struct Fp8Tile {
    uint32_t expert, first, rows;
};

// Row tiles of TILE rows of all groups, and the index-th of them; the same in every lane of the wave.
template <uint32_t TILE>
QMM_DEVICE uint32_t fp8_row_tiles(const Fp8Product& p) {
    if (!p.group_start) return (p.m + TILE - 1) / TILE;
    const uint32_t lane = threadIdx.x & 63;
    uint32_t total = 0;
    for (uint32_t e = lane; e < p.experts; e += 64)
        total += (fp8::group(p.group_start[e], p.group_start[e + 1], p.m).count + TILE - 1) / TILE;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) total += __shfl_xor(total, off, 64);
    return __builtin_amdgcn_readfirstlane(total);
}
template <uint32_t TILE>
QMM_DEVICE Fp8Tile fp8_row_tile(const Fp8Product& p, uint32_t index) {
    if (!p.group_start) return {0, index * TILE, min(p.m - index * TILE, TILE)};
    const uint32_t lane = threadIdx.x & 63;
    uint32_t before = 0;
    for (uint32_t e0 = 0; e0 < p.experts; e0 += 64) {
        const uint32_t e = e0 + lane;
        const fp8::Range g = e < p.experts ? fp8::group(p.group_start[e], p.group_start[e + 1], p.m) : fp8::Range{0, 0};
        const uint32_t tiles = (g.count + TILE - 1) / TILE;
        uint32_t sum = tiles;  // inclusive scan
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t u = __shfl_up(sum, d, 64);
            if (lane >= (uint32_t)d) sum += u;
        }
        const uint32_t start = before + sum - tiles;
        const uint64_t mine = __ballot(index >= start && index < start + tiles);
        if (mine) {
            const int at = __ffsll((unsigned long long)mine) - 1;
            const uint32_t i = index - __shfl(start, at, 64), first = __shfl(g.first, at, 64), count = __shfl(g.count, at, 64);
            return {(uint32_t)__builtin_amdgcn_readfirstlane(e0 + at), (uint32_t)__builtin_amdgcn_readfirstlane(first + i * TILE),
                    (uint32_t)__builtin_amdgcn_readfirstlane(min(count - i * TILE, TILE))};
        }
        before += __builtin_amdgcn_readfirstlane(__shfl(sum, 63, 64));
    }
    return {0, 0, 0};
}

stark_qmm_status launch_fp8_tiles(const Fp8Product& p, hipStream_t stream);

}  // namespace qmm
