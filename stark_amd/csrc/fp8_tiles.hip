// Tiles of products of 8-bit floating-point codes with block scales, dense or grouped by expert:
//   D[m, n] = sum_b (as[m, b] * bs[n / 128, b]) * sum_{k in b} A[m, k] B[n, k].
//
// A step is one block of 128 codes of the inner axis, whose sum of 16 x 16 outputs (fp8_block) starts at zero, is scaled in f32
// and added to the accumulator. The weights are the matrix instruction's rows, so that
// a lane's outputs are four consecutive columns of one row of D, and share one scale product.
#include "fp8_common.h"

namespace qmm {
namespace {

typedef __attribute__((address_space(3))) void lds_void;

constexpr uint32_t kStep = fp8::kBlock;  // codes (and bytes) of a row in a step

// LDS rows of 128 bytes, 16-byte piece c of row r at piece c ^ (r & 7): eight consecutive lanes of an operand read (rows
// r .. r + 7, one piece) and of a staging store cover the banks once.
template <int BM, int BN>
struct TileLds {
    u32x4 a[2][BM * 8];
    u32x4 b[2][BN * 8];
};

// Output tile of BM rows and BN columns by WM x WN waves.
template <int BM, int BN, int WM, int WN, bool EXACT>
__device__ __forceinline__ void fp8_tile(const Fp8Product& p, TileLds<BM, BN>& lds, const Fp8Tile t, uint32_t n0) {
    constexpr int W = WM * WN, MT = BM / WM / 16, NT = BN / WN / 16, LA = BM / 8 / W, LB = BN / 8 / W;
    static_assert(BM % (16 * WM) == 0 && BN % (16 * WN) == 0 && BM % (8 * W) == 0 && BN % (8 * W) == 0, "whole pieces a wave");
    static_assert(BN <= 128 || BN / WN <= 128, "one weight scale a wave and step");
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t wm = wave / WN, wn = wave % WN, col = lane & 15, kq = lane >> 4;
    const uint32_t steps = p.k / kStep, tail = p.k % kStep;

    // staging: a wave's i-th load takes rows 8 (i W + wave) .. + 7; rows past the tile's last are read from it
    const uint32_t srow = lane >> 3, piece = (lane & 7) ^ srow;
    const uint8_t* abase = p.a_rows ? p.a : p.a + (uint64_t)t.first * p.a_stride;
    const uint8_t* bbase = p.b + t.expert * p.b_expert + (uint64_t)n0 * p.b_stride;
    const uint32_t nlast = min((uint32_t)BN, p.n - n0) - 1;
    const auto a_row = [&](uint32_t r) {
        r = min(r, t.rows - 1);
        return p.a_rows ? min((uint32_t)p.a_rows[t.first + r], p.a_row_count - 1) : r;
    };
    uint32_t ao[LA], bo[LB];
#pragma unroll
    for (int i = 0; i < LA; ++i) ao[i] = a_row(8 * (i * W + wave) + srow) * (uint32_t)p.a_stride + 16 * piece;
#pragma unroll
    for (int i = 0; i < LB; ++i) bo[i] = min(8 * (i * W + wave) + srow, nlast) * (uint32_t)p.b_stride + 16 * piece;

    // scales: of the lane's row in each of its row blocks, and of the wave's columns
    const float* asbase = p.a_rows ? p.as : p.as + (uint64_t)t.first * p.as_row;
    const float* bsbase = p.bs + t.expert * p.bs_expert + (uint64_t)((n0 + wn * (BN / WN)) / kStep < fp8::blocks(p.n)
                                                                       ? (n0 + wn * (BN / WN)) / kStep : 0) * p.bs_row;
    uint32_t so[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) so[i] = a_row(wm * (BM / WM) + 16 * i + col) * (uint32_t)p.as_row;
    float sa[MT], sb;
    const auto load_scales = [&](uint32_t s) {
#pragma unroll
        for (int i = 0; i < MT; ++i) sa[i] = asbase[s * p.as_block + so[i]];
        sb = bsbase[s * p.bs_block];
    };

    const auto load = [&](uint32_t s, int buf) {
        const uint8_t* ab = abase + s * kStep;
        const uint8_t* bb = bbase + s * kStep;
#pragma unroll
        for (int i = 0; i < LA; ++i)
            __builtin_amdgcn_global_load_lds(ab + ao[i], (lds_void*)&lds.a[buf][64 * (i * W + wave)], 16, 0, 0);
#pragma unroll
        for (int i = 0; i < LB; ++i)
            __builtin_amdgcn_global_load_lds(bb + bo[i], (lds_void*)&lds.b[buf][64 * (i * W + wave)], 16, 0, 0);
    };
    // The last, short block: pieces past the row's end are not read, codes past it in its last piece are cleared.
    const auto load_tail = [&](int buf) {
        const uint32_t have = min(16u, tail > 16 * piece ? tail - 16 * piece : 0u);
        const auto cut = [&](const uint8_t* q) {
            u32x4 v = {0, 0, 0, 0};
            if (have) v = *(const u32x4*)q;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t n = have > 4u * e ? min(have - 4 * e, 4u) : 0;
                v[e] &= n == 4 ? 0xffffffffu : (1u << (8 * n)) - 1;
            }
            return v;
        };
#pragma unroll
        for (int i = 0; i < LA; ++i) lds.a[buf][64 * (i * W + wave) + lane] = cut(abase + steps * kStep + ao[i]);
#pragma unroll
        for (int i = 0; i < LB; ++i) lds.b[buf][64 * (i * W + wave) + lane] = cut(bbase + steps * kStep + bo[i]);
    };

    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

    const auto operand = [&](const u32x4* rows, uint32_t r) {
        const u32x4 x = rows[8 * r + ((2 * kq) ^ (r & 7))], y = rows[8 * r + ((2 * kq + 1) ^ (r & 7))];
        return Fp8Operand<EXACT>(i32x8{(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]});
    };
    const auto compute = [&](int buf, const float (&ca)[MT], float cb) {
        // (the operands of fewer columns at once where they are wide)
        constexpr int NC = EXACT ? 2 : NT;
#pragma unroll
        for (int j0 = 0; j0 < NT; j0 += NC) {
            Fp8Operand<EXACT> w[NC];
#pragma unroll
            for (int j = 0; j < NC; ++j) w[j] = operand(lds.b[buf], wn * (BN / WN) + 16 * (j0 + j) + col);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const auto x = operand(lds.a[buf], wm * (BM / WM) + 16 * i + col);
                const float s = ca[i] * cb;
#pragma unroll
                for (int j = 0; j < NC; ++j) {
                    const f32x4 v = fp8_block(w[j], x);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j0 + j][e] = fmaf(s, v[e], acc[i][j0 + j][e]);
                }
            }
        }
    };

    __syncthreads();  // a tile before this one may still be read
    int buf = 0;
    if (steps) load(0, 0);
    load_scales(0);
    for (uint32_t s = 0; s < steps; ++s) {
        __builtin_amdgcn_s_waitcnt(0xf70);  // vmcnt(0): this wave's pieces are in LDS
        __syncthreads();
        float ca[MT], cb = sb;
#pragma unroll
        for (int i = 0; i < MT; ++i) ca[i] = sa[i];
        if (s + 1 < steps) load(s + 1, buf ^ 1);
        if (s + 1 < steps || tail) load_scales(s + 1);
        compute(buf, ca, cb);
        buf ^= 1;
    }
    if (tail) {
        load_tail(buf);
        __syncthreads();
        compute(buf, sa, sb);
    }

    const void* bias = p.bias ? (const uint8_t*)p.bias + t.expert * p.bias_expert * (p.d_dt == STARK_QMM_F32 ? 4 : 2) : nullptr;
    // Outputs go through LDS, a row block at a time in the wave's own part, so that whole rows are stored.
    constexpr int C = BN / WN, P = C / 4 + 1;  // columns of the wave; pieces of a row, one more than it has: rows start on other banks
    static_assert(W * 16 * P <= 2 * 8 * (BM + BN), "the outputs' rows fit the operands' place");
    f32x4* const out = (f32x4*)&lds + wave * 16 * P;
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int k = 0; k < MT; ++k)
            if (i == k) {
#pragma unroll
                for (int j = 0; j < NT; ++j) out[col * P + 4 * j + kq] = acc[k][j];
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
        for (int j = 0; j < NT; ++j) {
            const uint32_t row = (64 * j + lane) / (C / 4), c = (64 * j + lane) % (C / 4), r = wm * (BM / WM) + 16 * i + row;
            if (r >= t.rows) continue;
            f32x4 v = out[row * P + c];
            if (p.a_rows && (uint32_t)p.a_rows[t.first + r] >= p.a_row_count) v = f32x4{1, 1, 1, 1} * __builtin_nanf("");
            fp8_store4(p, v, t.first + r, n0 + wn * C + 4 * c, bias);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

template <int BM, int BN, int WM, int WN, bool EXACT>
__global__ __launch_bounds__(64 * WM * WN) void fp8_tiles(Fp8Product p) {
    __shared__ TileLds<BM, BN> lds;
    const Fp8Groups<BM> groups(p);
    const uint32_t columns = (p.n + BN - 1) / BN, tiles = groups.total * columns;
    for (uint32_t i = blockIdx.x; i < (tiles + 7) / 8 * 8; i += gridDim.x) {
        const uint32_t t = fp8::tile_of(i, tiles);
        if (t >= tiles) continue;
        const Fp8Tile rows = groups.tile(p, t / columns);
        if (rows.rows) fp8_tile<BM, BN, WM, WN, EXACT>(p, lds, rows, (t % columns) * BN);
    }
}

template <int BM, int BN, int WM, int WN, bool EXACT>
stark_qmm_status launch(const Fp8Product& p, hipStream_t stream) {
    const uint64_t tiles = (uint64_t)fp8::row_tiles(p.m, p.experts, BM) * ((p.n + BN - 1) / BN);
    const uint32_t grid = (uint32_t)std::min<uint64_t>((tiles + 7) / 8 * 8, 1u << 20);
    hipLaunchKernelGGL((fp8_tiles<BM, BN, WM, WN, EXACT>), dim3(grid), dim3(64 * WM * WN), 0, stream, p);
    QMM_HIP_CHECK(hipGetLastError());
    return STARK_QMM_OK;
}

}  // namespace

stark_qmm_status launch_fp8_tiles(const Fp8Product& p, hipStream_t stream) {
    return p.d_dt == STARK_QMM_F32 ? launch<128, 128, 2, 2, true>(p, stream) : launch<128, 128, 2, 2, false>(p, stream);
}

}  // namespace qmm
