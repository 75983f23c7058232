// Rows to e4m3 with a scale for each 128 values: s = max(f32(max|x| / 448), 2^-126), codes the e4m3 values nearest to x / s.
//
// Sixteen lanes take a block, eight values each; the maximum is found over them by DPP. HBM bounds it: each value is read and
// each code written once (65536 gated rows of 768 in bf16 48.9 us, 5.2 TB/s; 8192 rows of 4096 23.3 us, 4.4 TB/s).
#include "fp8_common.h"

namespace qmm {
namespace {

constexpr int kThreads = 256, kLanes = 16;

struct Quantize {
    const void* x;
    uint8_t* codes;
    float* scales;
    const int32_t* row_count;
    uint64_t x_stride, code_stride, s_row, s_block;
    uint32_t rows, columns, blocks, inverse, items;
};

// Eight values of a row from column c on, as f32; zeros from column `end` on.
template <uint32_t DT, bool VEC>
QMM_DEVICE void load8(const void* x, uint64_t at, uint32_t c, uint32_t end, float (&v)[8]) {
    if (VEC && c + 8 <= end) {
        if constexpr (DT == STARK_QMM_F32) {
            const f32x4 a = *(const f32x4*)((const float*)x + at + c), b = *(const f32x4*)((const float*)x + at + c + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
        } else {
            const u32x4 t = *(const u32x4*)((const uint16_t*)x + at + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (DT == STARK_QMM_BF16) {
                    v[2 * e] = __uint_as_float(t[e] << 16), v[2 * e + 1] = __uint_as_float(t[e] & 0xffff0000u);
                } else {
                    v[2 * e] = f16_bits_to_f32(t[e] & 0xffffu), v[2 * e + 1] = f16_bits_to_f32(t[e] >> 16);
                }
            }
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < end ? load_as_f32(x, DT, at + c + e) : 0.0f;
}

// v * g / (1 + exp(-g)), the reciprocal to its last place; exp(-g) = 2^t with the product's rounding error carried into the result.
constexpr float kLog2e = 0x1.715476p+0f, kLog2eLow = 0x1.4ae0c0p-26f, kLn2 = 0x1.62e430p-1f;
QMM_DEVICE float gate(float v, float g) {
    const float t = -g * kLog2e, r = fmaf(-g, kLog2eLow, fmaf(-g, kLog2e, -t));
    const float p = __builtin_amdgcn_exp2f(t), ex = fabsf(t) < 128.0f ? fmaf(p, r * kLn2, p) : p;
    return v * (g * __builtin_amdgcn_rcpf(1.0f + ex));
}

// The same below kFarGate, where 1 + exp(-g) nears f32's end, its reciprocal is subnormal (v_rcp_f32 gives zero) and then exp(-g)
// infinite: the sigmoid is exp(g), as four equal factors, so that nothing but the product itself leaves the normal range.
constexpr float kFarGate = -87.0f;
QMM_DEVICE float gate_far(float v, float g) {
    const float t = g * kLog2e, r = fmaf(g, kLog2eLow, fmaf(g, kLog2e, -t)), q = __builtin_amdgcn_exp2f(0.25f * t);
    return v * q * q * q * (g * q) * (t > -512.0f ? fmaf(r, kLn2, 1.0f) : 1.0f);
}

// e4m3 codes of x[0] / s and x[1] / s in the low 16 bits; i is within a few ulp of 1 / s. Where the quotient is so near the
// middle of two codes that its error may matter, the sign of middle * s - x, which an fma gives exactly, decides.
QMM_DEVICE uint32_t codes2(float x0, float x1, float s, float i) {
    const float q0 = fminf(fmaxf(x0 * i, -448.0f), 448.0f), q1 = fminf(fmaxf(x1 * i, -448.0f), 448.0f);
    constexpr float kDown = 1.0f - 0x1p-20f, kUp = 1.0f + 0x1p-20f;
    uint32_t lo = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q0 * kDown, q1 * kDown, 0, false) & 0xffffu;
    const uint32_t hi = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(fminf(fmaxf(q0 * kUp, -448.0f), 448.0f),
                                                                  fminf(fmaxf(q1 * kUp, -448.0f), 448.0f), 0, false) & 0xffffu;
    if (lo != hi) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t a = (lo >> (8 * e)) & 255u, b = (hi >> (8 * e)) & 255u;
            if (a == b) continue;
            const float x = e ? fabsf(x1) : fabsf(x0);
            const float middle = 0.5f * (__builtin_amdgcn_cvt_f32_fp8(a & 127u, 0) + __builtin_amdgcn_cvt_f32_fp8(b & 127u, 0));
            const float up = s < 1.0f ? 0x1p64f : 1.0f;  // no difference is lost below the smallest f32
            const float d = fmaf(middle, s * up, -(x * up));
            const uint32_t c = d > 0.0f ? a : d < 0.0f ? b : (a & 1u) ? b : a;
            lo = e ? (lo & 0x00ffu) | (c << 8) : (lo & 0xff00u) | c;
        }
    }
    return lo;
}

template <uint32_t DT, bool GATED, bool VEC>
__global__ __launch_bounds__(kThreads) void fp8_quantize(Quantize q) {
    const uint32_t item = blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
    const fp8::Split at = fp8::split(min(item, q.items - 1), q.blocks, q.inverse);
    const uint32_t rows = q.row_count ? (uint32_t)min(max(*q.row_count, 0), (int32_t)q.rows) : q.rows;
    if (item >= q.items || at.row >= rows) return;  // whole groups of sixteen lanes leave
    const uint64_t x_at = at.row * q.x_stride;
    const uint32_t c = at.block * fp8::kBlock + 8 * lane;
    float v[8];
    load8<DT, VEC>(q.x, x_at, c, q.columns, v);
    if constexpr (GATED) {
        float g[8];
        load8<DT, VEC>(q.x, x_at + q.columns, c, q.columns, g);
        uint32_t low = 0;  // the lowest gate's bits: those of negative values are above the others', and the higher the lower the value
#pragma unroll
        for (int e = 0; e < 8; ++e) low = max(low, __float_as_uint(g[e]));
        if (low > __float_as_uint(kFarGate)) {  // (a branch around the eight: 65536 rows of 768 in bf16 48.9 us, with a choice for each value 50.6)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = g[e] < kFarGate ? gate_far(v[e], g[e]) : gate(v[e], g[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = gate(v[e], g[e]);
        }
    }
    uint32_t top = 0;  // the largest magnitude's bits: those of a NaN are above an infinity's, and these above the rest
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    top = group_max<kLanes>(top);
    const bool bad = top >= 0x7f800000u;
    const float s = fmaxf(__uint_as_float(bad ? 0 : top) / 448.0f, 0x1p-126f), i = __builtin_amdgcn_rcpf(s);
    uint32_t w[2] = {0, 0};
    if (!bad) {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e / 2] |= codes2(v[2 * e], v[2 * e + 1], s, i) << (16 * (e % 2));
    }
    uint8_t* out = q.codes + at.row * q.code_stride + c;
    if (c + 8 <= q.columns) {
        *(uint2*)out = uint2{w[0], w[1]};
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < q.columns) out[e] = (uint8_t)(w[e / 4] >> (8 * (e % 4)));
    }
    if (lane == 0) q.scales[at.row * q.s_row + at.block * q.s_block] = bad ? __builtin_nanf("") : s;
}

template <uint32_t DT>
void launch(const Quantize& q, bool gated, bool vec, hipStream_t s) {
    const dim3 grid((q.items + kThreads / kLanes - 1) / (kThreads / kLanes)), block(kThreads);
    if (gated) {
        if (vec) hipLaunchKernelGGL((fp8_quantize<DT, true, true>), grid, block, 0, s, q);
        else hipLaunchKernelGGL((fp8_quantize<DT, true, false>), grid, block, 0, s, q);
    } else {
        if (vec) hipLaunchKernelGGL((fp8_quantize<DT, false, true>), grid, block, 0, s, q);
        else hipLaunchKernelGGL((fp8_quantize<DT, false, false>), grid, block, 0, s, q);
    }
}

}  // namespace
}  // namespace qmm

extern "C" stark_qmm_status stark_qmm_fp8_quantize(const stark_qmm_fp8_quantize_args* a, void* stream) {
    using namespace qmm;
    if (!a) return STARK_QMM_INVALID_ARGUMENT;
    if (a->struct_size != sizeof(*a)) return STARK_QMM_ABI_MISMATCH;
    if (!fp8_type(a->data_type)) return STARK_QMM_UNSUPPORTED_DATA_TYPE;
    if (a->rows > (1u << 24) || a->columns > (1u << 20)) return STARK_QMM_INVALID_ARGUMENT;
    if (a->rows == 0 || a->columns == 0) return STARK_QMM_OK;
    const uint64_t e = fp8_element(a->data_type), wide = (uint64_t)a->columns * (a->gated ? 2 : 1), rows = a->rows;
    const uint32_t blocks = fp8::blocks(a->columns);
    // a launch has fewer than 2^32 threads, whole workgroups of them: sixteen blocks each
    if (rows * blocks > (1ull << 28) - kThreads / kLanes) return STARK_QMM_UNSUPPORTED;
    if (!a->x || !a->codes || !a->scales || !fp8_aligned(a->x, e) || !fp8_aligned(a->codes, 16) || !fp8_aligned(a->scales, 4) ||
        !fp8_aligned(a->row_count, 4))
        return STARK_QMM_INVALID_ARGUMENT;
    if ((a->x_row_stride | a->code_row_stride | a->scale_row_stride | a->scale_block_stride) >> 40) return STARK_QMM_INVALID_ARGUMENT;
    if (rows > 1 && (a->x_row_stride < wide || a->code_row_stride < a->columns || a->code_row_stride % 16)) return STARK_QMM_INVALID_ARGUMENT;
    const uint64_t xs = rows > 1 ? a->x_row_stride : 0, cs = rows > 1 ? a->code_row_stride : 0, ss = rows > 1 ? a->scale_row_stride : 0;
    // distinct scales: blocks inside rows, or rows inside blocks
    const uint64_t sb = blocks > 1 ? a->scale_block_stride : 0;
    if (!((blocks == 1 || sb >= 1) && (rows == 1 || ss >= 1) &&
          (rows == 1 || blocks == 1 || ss >= (blocks - 1) * sb + 1 || sb >= (rows - 1) * ss + 1)))
        return STARK_QMM_INVALID_ARGUMENT;
    const uint64_t xn = e * fp8_span(rows, xs, wide), cn = fp8_span(rows, cs, a->columns), sn = 4 * (fp8_span(rows, ss, 1) + (blocks - 1) * sb);
    if (fp8_overlap(a->codes, cn, a->x, xn) || fp8_overlap(a->scales, sn, a->x, xn) || fp8_overlap(a->codes, cn, a->scales, sn) ||
        fp8_overlap(a->row_count, 4, a->codes, cn) || fp8_overlap(a->row_count, 4, a->scales, sn))
        return STARK_QMM_INVALID_ARGUMENT;
    Quantize q{a->x, a->codes, a->scales, a->row_count, xs, cs, ss, sb, a->rows, a->columns, blocks, fp8::inverse(blocks), (uint32_t)(rows * blocks)};
    // rows (and gates) that start on 16-byte boundaries are read in pieces
    const bool vec = fp8_aligned(a->x, 16) && xs * e % 16 == 0 && (!a->gated || a->columns * e % 16 == 0);
    if (a->data_type == STARK_QMM_F32) launch<STARK_QMM_F32>(q, a->gated, vec, (hipStream_t)stream);
    else if (a->data_type == STARK_QMM_F16) launch<STARK_QMM_F16>(q, a->gated, vec, (hipStream_t)stream);
    else launch<STARK_QMM_BF16>(q, a->gated, vec, (hipStream_t)stream);
    QMM_HIP_CHECK(hipGetLastError());
    return STARK_QMM_OK;
}
