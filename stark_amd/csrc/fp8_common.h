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
    uint32_t first_group;  // workgroup of the call that a launch's first one is (among the sizes, which are loaded first: at the
                           // end grouped decode took 44.4 us instead of 43.4)
    uint32_t d_dt, flags;
    float ab_scale, soft_cap;
    uint32_t vec;    // four outputs of a row may be stored at once
    uint32_t plain;  // eight 16-bit ones, that are the scaled sums
    uint32_t parts;  // runs of the inner axis, whose sums meet in `partial` [parts, m, partial_stride]
    float* partial;
    uint64_t partial_stride;
};

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Bytes of two row ranges [rows, width] (width and stride in bytes) meet.
inline bool fp8_overlap(const void* p, uint64_t pn, const void* q, uint64_t qn) {
    return p && q && pn && qn && (uintptr_t)p < (uintptr_t)q + qn && (uintptr_t)q < (uintptr_t)p + pn;
}
inline uint64_t fp8_span(uint64_t rows, uint64_t stride, uint64_t width) { return rows ? (rows - 1) * stride + width : 0; }
// A call's workgroups in as many launches as they need.
template <typename Launch>
stark_qmm_status fp8_launch(Fp8Product p, uint64_t groups, uint32_t threads, const Launch& launch) {
    const uint32_t most = fp8::launch_groups(threads);
    for (uint64_t first = 0; first < groups; first += most) {
        p.first_group = (uint32_t)first;
        launch(p, (uint32_t)std::min<uint64_t>(groups - first, most));
        QMM_HIP_CHECK(hipGetLastError());
    }
    return STARK_QMM_OK;
}
inline bool fp8_aligned(const void* p, uint64_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
inline uint64_t fp8_element(uint32_t dt) { return dt == STARK_QMM_F32 ? 4 : 2; }
inline bool fp8_exact(uint32_t d_dt) { return d_dt != STARK_QMM_BF16; }  // sums of f32 (Fp8Operand)
inline bool fp8_type(uint32_t dt) { return dt == STARK_QMM_F32 || dt == STARK_QMM_F16 || dt == STARK_QMM_BF16; }

// A 16 x 16 block of A B over 128 codes, from zero: lane l has row (column) l % 16 of A (B) and 32 of its codes (which 32 does
// not matter while both operands agree), and outputs (4 (l / 16) + e, l % 16).
//
// v_mfma_f32_16x16x128_f8f6f4 takes codes as they are. It adds products in groups of eight neighbouring codes, and what a
// product has below 2^-13 of the largest product's binade in its group is cut off before the sum (measured; sums of groups are
// f32): outputs of normally distributed codes are off by 1.5e-5 of the outputs' norm. bf16 outputs take it, whose own rounding is
// off by 1.7e-3. f16 and f32 ones would show it (an f16 output of a tenth of the norm is rounded by 2e-5 of it): their codes are
// widened to bf16 first, exactly, and v_mfma_f32_16x16x32_bf16 adds in f32 (1e-8), at half the rate.
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

// Two outputs in 16 bits.
typedef __bf16 fp8_bf16x2 __attribute__((ext_vector_type(2)));
QMM_DEVICE uint32_t fp8_pack2(uint32_t dt, float a, float b) {
    if (dt == STARK_QMM_BF16) return __builtin_bit_cast(uint32_t, fp8_bf16x2{(__bf16)a, (__bf16)b});
    return f32_to_f16_bits(a) | (uint32_t)f32_to_f16_bits(b) << 16;
}

// Four consecutive outputs of a row from column n on.
QMM_DEVICE void fp8_store4(const Fp8Product& p, f32x4 sum, uint32_t row, uint32_t n, const void* bias) {
    const size_t at = (size_t)row * p.d_stride + n;
    if (n >= p.n) return;
    if (!p.vec || n + 4 > p.n) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < p.n) store_from_f32(p.d, p.d_dt, at + e, fp8_finish(p, sum[e], at + e, bias, n + e));
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

// Sum over the lanes up to and with this one.
QMM_DEVICE uint32_t fp8_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
    return v;
}

// The groups of a call as one wave sees them: lane l has up to sixteen consecutive ones, all loaded at once.
template <uint32_t TILE>
struct Fp8Groups {
    static constexpr uint32_t kEach = 16;  // 64 lanes, 1024 groups
    int32_t start[kEach + 1];
    uint32_t each, total, before, mine;  // groups a lane; row tiles of all, of the lanes before this one, of this one

    QMM_DEVICE static uint32_t tiles(fp8::Range g) { return (g.count + TILE - 1) / TILE; }

    QMM_DEVICE explicit Fp8Groups(const Fp8Product& p) {
        if (!p.group_start) {
            total = (p.m + TILE - 1) / TILE;
            return;
        }
        const uint32_t lane = threadIdx.x & 63;
        each = (p.experts + 63) / 64;
#pragma unroll
        for (uint32_t i = 0; i <= kEach; ++i)
            if (i <= each) start[i] = p.group_start[min(lane * each + i, p.experts)];
        mine = 0;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i)
            if (i < each) mine += tiles(fp8::group(start[i], start[i + 1], p.m));
        const uint32_t sum = fp8_scan(mine);
        before = sum - mine;
        total = (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
    }

    // The index-th row tile; the same in every lane.
    QMM_DEVICE Fp8Tile tile(const Fp8Product& p, uint32_t index) const {
        if (!p.group_start) return {0, index * TILE, index < total ? min(p.m - index * TILE, TILE) : 0};
        const uint64_t found = __ballot(index - before < mine);
        if (!found) return {0, 0, 0};
        const int at = __ffsll((unsigned long long)found) - 1;
        uint32_t i = index - (uint32_t)__builtin_amdgcn_readlane((int)before, at);
        Fp8Tile t{0, 0, 0};
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) {
            if (e >= each || t.rows) continue;
            const fp8::Range g = fp8::group(__builtin_amdgcn_readlane(start[e], at), __builtin_amdgcn_readlane(start[e + 1], at), p.m);
            if (i < tiles(g)) t = Fp8Tile{at * each + e, g.first + i * TILE, min(g.count - i * TILE, TILE)};
            else i -= tiles(g);
        }
        return t;
    }
};

stark_qmm_status launch_fp8_rows(const Fp8Product& p, uint32_t rows, hipStream_t stream);
stark_qmm_status launch_fp8_tiles(const Fp8Product& p, uint32_t tile, hipStream_t stream);

}  // namespace qmm
