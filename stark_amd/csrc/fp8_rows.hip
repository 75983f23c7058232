// Products of 8-bit floating-point codes with few rows, dense or grouped by expert: the weights are read once, from memory
// straight into registers.
//
// A workgroup takes a strip of 16 NT columns and up to 16 MT rows (16, or 32 by 32 columns); its W waves share the inner axis, in
// runs of whole blocks, and their sums meet in LDS, in wave order. HBM bounds it: one row, N 12288, K 4096 10.6 us (4.7 TB/s, the
// launch within), 16 tokens on 8 of 128 experts, N 1536, K 2048 43.2 us (5.25 TB/s); with more rows the reads of their codes by
// every workgroup do (N 4096, K 12288, five rows 12.3 us, in f16 with a bias 13.1; 16 rows 14.1).
#include "fp8_common.h"

namespace qmm {
namespace {

// Bytes of a piece that starts at byte `at` of a row of k codes, those past its end cleared.
QMM_DEVICE void cut_piece(u32x4& v, uint32_t at, uint32_t k) {
    const uint32_t have = at < k ? min(k - at, 16u) : 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t n = have > 4u * e ? min(have - 4 * e, 4u) : 0;
        v[e] &= n == 4 ? 0xffffffffu : (1u << (8 * n)) - 1;
    }
}

template <int MT, int NT, int W, bool EXACT>
__global__ __launch_bounds__(64 * W) void fp8_rows(Fp8Product p) {
    // blocks of a wave whose loads are in flight
    constexpr int S = NT == 1 ? 4 : 2;
    __shared__ f32x4 sums[W][MT][NT][64];
    const uint32_t tid = threadIdx.x, lane = tid & 63, col = lane & 15, kq = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t strips = (p.n + 16 * NT - 1) / (16 * NT), blocks = fp8::blocks(p.k);
    const uint32_t each = (blocks + W - 1) / W, b0 = min(wave * each, blocks), b1 = min(b0 + each, blocks);
    const uint32_t group = p.first_group + blockIdx.x;
    const Fp8Tile t = Fp8Groups<16 * MT>(p).tile(p, group / strips);
    if (!t.rows) return;
    const uint32_t n0 = (group % strips) * 16 * NT;

    uint32_t ar[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        ar[j] = t.first + min(16u * j + col, t.rows - 1);
        if (p.a_rows) ar[j] = min((uint32_t)p.a_rows[ar[j]], p.a_row_count - 1);
    }
    // A load instruction takes whole 128-byte lines of eight rows: lane l piece 2 (l / 16) + (l / 8) % 2 of row l % 8, then, the
    // other way round, of row 8 + l % 8. So a lane has one piece of its own row and one of its neighbour's, eight lanes on.
    const uint8_t* b = p.b + t.expert * p.b_expert;
    const uint8_t* wp[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        wp[j][0] = b + (uint64_t)min(n0 + 16 * j + (lane & 7), p.n - 1) * p.b_stride;
        wp[j][1] = b + (uint64_t)min(n0 + 16 * j + 8 + (lane & 7), p.n - 1) * p.b_stride;
    }
    const uint32_t w_at[2] = {16 * (2 * kq + ((lane >> 3) & 1)), 16 * (2 * kq + 1 - ((lane >> 3) & 1))};
    const uint32_t last_piece = (p.k - 1) / 16 * 16;  // pieces past a row's last are read from it, and cleared
    const float* bs = p.bs + t.expert * p.bs_expert + (uint64_t)(n0 / fp8::kBlock) * p.bs_row;

    u32x4 wv[S][NT][2], av[S][MT][2];
    float sa[S][MT], sb[S];
    const auto load_weights = [&](int u, uint32_t c) {
        const uint32_t k0 = c * fp8::kBlock;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) wv[u][j][h] = *(const u32x4*)(wp[j][h] + min(k0 + w_at[h], last_piece));
        sb[u] = bs[c * p.bs_block];
    };
    const auto load_rows = [&](int u, uint32_t c) {
        const uint32_t k0 = c * fp8::kBlock;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const uint8_t* a = p.a + (uint64_t)ar[m] * p.a_stride;
#pragma unroll
            for (int h = 0; h < 2; ++h) av[u][m][h] = *(const u32x4*)(a + min(k0 + 32 * kq + 16 * h, last_piece));
            sa[u][m] = p.as[ar[m] * p.as_row + c * p.as_block];
        }
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[m][j] = f32x4{0, 0, 0, 0};
    const auto compute = [&](int u, uint32_t c) {
        const uint32_t k0 = c * fp8::kBlock;
        if (k0 + fp8::kBlock > p.k) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int j = 0; j < NT; ++j) cut_piece(wv[u][j][h], k0 + w_at[h], p.k);
#pragma unroll
                for (int m = 0; m < MT; ++m) cut_piece(av[u][m][h], k0 + 32 * kq + 16 * h, p.k);
            }
        }
        Fp8Operand<EXACT> w[NT];
        const bool high = lane & 8;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            i32x8 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t x = wv[u][j][0][e], y = wv[u][j][1][e];
                v[e] = (int)(high ? y : x);
                v[4 + e] = __builtin_amdgcn_update_dpp(0, (int)(high ? x : y), 0x128, 0xf, 0xf, false);  // row_ror:8
            }
            w[j] = Fp8Operand<EXACT>(v);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const u32x4 x = av[u][m][0], y = av[u][m][1];
            const Fp8Operand<EXACT> a(i32x8{(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]});
            const float s = sa[u][m] * sb[u];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const f32x4 v = fp8_block(w[j], a);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[m][j][e] = fmaf(s, v[e], acc[m][j][e]);
            }
        }
    };
    if (b0 < b1) {
#pragma unroll
        for (int u = 0; u < S; ++u) load_weights(u, min(b0 + u, b1 - 1));
#pragma unroll
        for (int u = 0; u < S; ++u) load_rows(u, min(b0 + u, b1 - 1));
        uint32_t c = b0;
        for (; c + S < b1; c += S) {
#pragma unroll
            for (int u = 0; u < S; ++u) {
                compute(u, c + u);
                // (past the run's end its last block again, out of the caches: a load less on one way into a wait would make
                // it wait for more on the other)
                load_weights(u, min(c + u + S, b1 - 1));
                load_rows(u, min(c + u + S, b1 - 1));
            }
        }
#pragma unroll
        for (int u = 0; u < S; ++u)
            if (c + u < b1) compute(u, c + u);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j) sums[wave][m][j][lane] = acc[m][j];
    __syncthreads();
    const void* bias = p.bias ? (const uint8_t*)p.bias + t.expert * p.bias_expert * (p.d_dt == STARK_QMM_F32 ? 4 : 2) : nullptr;
    for (uint32_t o = tid; o < 64 * MT * NT; o += 64 * W) {
        const uint32_t m = o / (64 * NT), j = o / 64 % NT, l = o % 64, r = 16 * m + (l & 15);
        f32x4 v = sums[0][m][j][l];
#pragma unroll
        for (int w = 1; w < W; ++w) v += sums[w][m][j][l];
        if (r >= t.rows) continue;
        if (p.a_rows && (uint32_t)p.a_rows[t.first + r] >= p.a_row_count) v = f32x4{1, 1, 1, 1} * __builtin_nanf("");
        fp8_store4(p, v, t.first + r, n0 + 16 * j + 4 * (l >> 4), bias);
    }
}

template <int MT, int NT, int W>
stark_qmm_status launch(const Fp8Product& p, hipStream_t stream) {
    const uint64_t tiles = (uint64_t)fp8::row_tiles(p.m, p.experts, 16 * MT) * ((p.n + 16 * NT - 1) / (16 * NT));
    return fp8_launch(p, tiles, 64 * W, [&](const Fp8Product& part, uint32_t groups) {
        if (fp8_exact(p.d_dt)) hipLaunchKernelGGL((fp8_rows<MT, NT, W, true>), dim3(groups), dim3(64 * W), 0, stream, part);
        else hipLaunchKernelGGL((fp8_rows<MT, NT, W, false>), dim3(groups), dim3(64 * W), 0, stream, part);
    });
}

}  // namespace

stark_qmm_status launch_fp8_rows(const Fp8Product& p, uint32_t rows, hipStream_t stream) {
    const uint64_t tiles = fp8::row_tiles(p.m, p.experts, rows);
    if (rows == 32) return tiles * ((p.n + 31) / 32) < 256 ? launch<2, 2, 8>(p, stream) : launch<2, 2, 4>(p, stream);
    const fp8::RowShare s = fp8::row_share(tiles, p.n, p.k);
    if (s.strips == 2) return launch<1, 2, 4>(p, stream);
    if (s.waves <= 2) return launch<1, 1, 2>(p, stream);
    if (s.waves <= 4) return launch<1, 1, 4>(p, stream);
    return s.waves <= 8 ? launch<1, 1, 8>(p, stream) : launch<1, 1, 16>(p, stream);
}

}  // namespace qmm
