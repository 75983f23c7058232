// Tiles of products of 8-bit floating-point codes with block scales, dense or grouped by expert:
//   D[m, n] = sum_b (as[m, b] * bs[n / 128, b]) * sum_{k in b} A[m, k] B[n, k].
//
// A step is one block of 128 codes of the inner axis, whose sum of 16 x 16 outputs (fp8_block) starts at zero, is scaled in f32
// and added to the accumulator. The weights are the matrix instruction's rows, so that a lane's outputs are four consecutive
// columns of one row of D, and share one scale product. Operands go from memory into LDS without registers between.
//
// 256 x 256 outputs by eight waves (64 x 128 each): 64 rows and 128 columns of a wave are 24 LDS reads for 32 matrix instructions,
// so that LDS is busy for half of their time, and the tile reads half of what 128 x 128 tiles read. 4096 rows, N 12288, K 4096 take
// 190 us (2170 TFLOP/s; a large product with one scale a tensor reaches 2660 on this card). The matrix instructions bound it
// (82 us at their peak), with the starts of steps, where two waves a SIMD wait for their operands out of LDS, and the start and
// the stores of a tile, some 8 us that nothing hides: one workgroup to a CU. (A version of 222 us took 97 with its loads alone,
// 141 with its products alone and 173 without its stores.) 65536 rows of 128 experts, N 1536, K 2048, whose tiles have 16 steps:
// 292 us. Steps on the way to it, for the first call: 128 x 128 tiles with a lane's scales loaded each step 382 us; 256 x 256 274;
// scales staged 228; LDS pieces without conflicts 223; outputs from registers 203; a scalar step offset and the order of the
// products held 188. 128 x 128 by four waves (two workgroups to a CU) takes smaller calls, 64 x 64 with three steps in LDS the
// smallest, where each step is latency (0.35 us). Sums of f32 (f16 and f32 outputs) widen the codes on the way to the matrix
// instruction and take 128 x 128 at most: the first call in f16 364 to 372 us.
#include "fp8_common.h"

namespace qmm {
namespace {

typedef __attribute__((address_space(3))) void lds_void;

constexpr uint32_t kStep = fp8::kBlock;  // codes (and bytes) of a row in a step

// What a 32-bit offset reaches from p on: the offsets here stay inside the operands by themselves.
QMM_DEVICE __amdgpu_buffer_rsrc_t everything(const void* p) { return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, 0xffffffff, 0x00020000); }

constexpr uint32_t kChunk = 8;  // steps whose scales of the rows are staged together

// LDS rows of 128 bytes, 16-byte piece c of row r at piece c ^ (r / 2 % 8). Sixteen lanes of an operand read cover the 64 banks
// once, be they lanes with one piece of sixteen rows or, as a 16-byte read takes them, four lanes each of rows r and r + 12 with
// piece c and of r + 4 and r + 8 with piece c + 1.
template <int BM, int BN, int W, int S>
struct TileLds {
    u32x4 a[S][BM * 8];
    u32x4 b[S][BN * 8];
    float sa[2][BM * kChunk];  // [8 rows][step][row] of a chunk
    float sb[2][64];           // [128 columns][step]
};

// Output tile of BM rows and BN columns by WM x WN waves, with the operands of S steps in LDS; the `part`-th of p.parts runs of
// the steps.
template <int BM, int BN, int WM, int WN, int S, bool EXACT>
__device__ __forceinline__ void fp8_tile(const Fp8Product& p, TileLds<BM, BN, WM * WN, S>& lds, const Fp8Tile t, uint32_t n0, uint32_t part) {
    constexpr int W = WM * WN, MT = BM / WM / 16, NT = BN / WN / 16, LA = BM / 8 / W, LB = BN / 8 / W;
    static_assert(BM % (16 * WM) == 0 && BN % (16 * WN) == 0 && BM % (8 * W) == 0 && BN % (8 * W) == 0, "whole pieces a wave");
    static_assert(BN <= 128 || BN / WN <= 128, "one weight scale a wave and step");
    static_assert(W % 2 == 0, "a wave's staged rows have one swizzle");
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t wm = wave / WN, wn = wave % WN, col = lane & 15, kq = lane >> 4;
    const uint32_t steps = p.k / kStep, tail = p.k % kStep;
    const uint32_t before = tail ? 1 : 0, all = steps + before;  // a short last block is the first step
    const uint32_t from = part * all / p.parts, total = (part + 1) * all / p.parts;

    // staging: a wave's i-th load takes rows 8 (i W + wave) .. + 7; rows past the tile's last are read from it
    const uint32_t srow = lane >> 3, piece = (lane & 7) ^ ((4 * wave + (srow >> 1)) & 7);
    const uint8_t* abase = p.a_rows ? p.a : p.a + (uint64_t)t.first * p.a_stride;
    const uint8_t* bbase = p.b + t.expert * p.b_expert + (uint64_t)n0 * p.b_stride;
    const uint32_t nlast = min((uint32_t)BN, p.n - n0) - 1;
    const auto a_row = [&](uint32_t r) {
        r = min(r, t.rows - 1);
        return p.a_rows ? min((uint32_t)p.a_rows[t.first + r], p.a_row_count - 1) : r;
    };
    // (rows and scales first: gathered ones are loads of their own, which the weights' first loads need not wait for)
    uint32_t ao[LA], bo[LB], so[LA];
#pragma unroll
    for (int i = 0; i < LA; ++i) ao[i] = a_row(8 * (i * W + wave) + srow);
#pragma unroll
    for (int i = 0; i < LA; ++i) so[i] = a_row(8 * (i * W + wave) + (lane & 7));
#pragma unroll
    for (int i = 0; i < LB; ++i) bo[i] = min(8 * (i * W + wave) + srow, nlast) * (uint32_t)p.b_stride + 16 * piece;

    const __amdgpu_buffer_rsrc_t ra = everything(abase), rb = everything(bbase);
    const auto load_b = [&](uint32_t s, int buf) {  // a step that is not the short one
        const uint32_t k0 = __builtin_amdgcn_readfirstlane((s - before) * kStep);
#pragma unroll
        for (int i = 0; i < LB; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_void*)&lds.b[buf][64 * (i * W + wave)], 16, bo[i], k0, 0, 0);
    };
    const auto load_a = [&](uint32_t s, int buf) {
        const uint32_t k0 = __builtin_amdgcn_readfirstlane((s - before) * kStep);
#pragma unroll
        for (int i = 0; i < LA; ++i)
            if (S > 2 || 8 * (i * W + wave) < t.rows)  // (with S > 2 a wave's loads of a step are counted)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_void*)&lds.a[buf][64 * (i * W + wave)], 16, ao[i], k0, 0, 0);
    };
    if (from >= before && from < total) load_b(from, 0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < LA; ++i) ao[i] = ao[i] * (uint32_t)p.a_stride + 16 * piece, so[i] *= (uint32_t)p.as_row;
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
    // Scales of a chunk of steps: a load takes eight rows' (one line each where a row's scales are contiguous).
    const float* asbase = p.a_rows ? p.as : p.as + (uint64_t)t.first * p.as_row;
    const float* bsbase = p.bs + t.expert * p.bs_expert;
    const auto load_scales = [&](uint32_t chunk) {
        const auto block = [&](uint32_t in) {
            const uint32_t s = min(from + chunk * kChunk + in, total - 1);
            return s < before ? steps : s - before;
        };
        const uint32_t s = block(lane >> 3);
#pragma unroll
        for (int i = 0; i < LA; ++i)
            __builtin_amdgcn_global_load_lds(asbase + s * p.as_block + so[i], (lds_void*)&lds.sa[chunk & 1][64 * (i * W + wave)], 4, 0, 0);
        if (wave == 0) {
            const uint32_t nb = min(n0 / kStep + (lane >> 3), fp8::blocks(p.n) - 1), sl = block(lane & 7);
            __builtin_amdgcn_global_load_lds(bsbase + nb * p.bs_row + sl * p.bs_block, (lds_void*)&lds.sb[chunk & 1][0], 4, 0, 0);
        }
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

    const uint32_t p0 = 8 * col + (kq ^ (col >> 1)), p1 = p0 ^ 4;  // pieces kq and kq + 4
    const auto operand = [&](const u32x4* rows) {  // 16 rows from `rows` on
        const u32x4 x = rows[p0], y = rows[p1];
        return Fp8Operand<EXACT>(i32x8{(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]});
    };
    const auto compute = [&](int buf, uint32_t s) {
        const uint32_t in = (s - from) % kChunk, cb = (s - from) / kChunk & 1;
        // A matrix instruction's result takes some twelve issue slots: each sum is scaled two instructions later, and the
        // columns' codes are read two column blocks ahead. The order is held as it is written: the first instruction waits for its
        // own operands only, the scales come last.
        constexpr int D = 2, Q = MT * NT;
        f32x4 v[D + 1];
        Fp8Operand<EXACT> w[2], x[MT];
        float c[MT];
        const auto columns = [&](int j) { return operand(lds.b[buf] + 8 * (wn * (BN / WN) + 16 * j)); };
        w[0] = columns(0);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            x[i] = operand(lds.a[buf] + 8 * (wm * (BM / WM) + 16 * i));
            if (!EXACT) __builtin_amdgcn_sched_barrier(0);
        }
        if (NT > 1) w[1] = columns(1);
        if (!EXACT) __builtin_amdgcn_sched_barrier(0);
        const float sb = lds.sb[cb][8 * (wn * (BN / WN) / kStep) + in];
#pragma unroll
        for (int i = 0; i < MT; ++i) c[i] = lds.sa[cb][8 * (wm * (BM / WM) + 16 * i) + 64 * (col >> 3) + 8 * in + (col & 7)];
        if (!EXACT) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < Q + D; ++q) {
            if (q < Q) v[q % (D + 1)] = fp8_block(w[q / MT % 2], x[q % MT]);
            if (!EXACT) __builtin_amdgcn_sched_barrier(0);
            if (q == D - 1) {
#pragma unroll
                for (int i = 0; i < MT; ++i) c[i] *= sb;
            }
            if (q >= D) {
                const int i = (q - D) % MT, j = (q - D) / MT;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(c[i], v[(q - D) % (D + 1)][e], acc[i][j][e]);
            }
            if (q < Q && q % MT == MT - 1 && q / MT + 2 < NT) w[q / MT % 2] = columns(q / MT + 2);
            if (!EXACT) __builtin_amdgcn_sched_barrier(0);
        }
    };

    // A step's loads are issued S - 1 steps ahead and waited for at its start, while those of the steps between stay in flight:
    // where a wave passes the barrier, all waves' pieces are in LDS and none still reads the buffer that is loaded next. (No
    // fence here: one would wait for all loads.)
    constexpr int F = (S - 2) * (LA + LB);  // loads of the steps between
    const auto arrive = [&](bool between) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        if (S > 2 && between) __builtin_amdgcn_s_waitcnt(0x0070 | (F & 15) | (F >> 4 << 14));  // vmcnt(F), lgkmcnt(0)
        else __builtin_amdgcn_s_waitcnt(0x0070);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
    };
    load_scales(0);
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
        if (from + i < total) {
            if (from + i < before) {
                load_tail(i);
            } else {
                load_a(from + i, i);
                if (i > 0) load_b(from + i, i);
            }
        }
    int buf = 0;
#pragma unroll 1
    for (uint32_t s = from; s < total; ++s) {
        arrive(s + S - 2 < total);
        if (s + S - 1 < total) {
            const uint32_t next = s + S - 1 - from;
            if (next % kChunk == 0) load_scales(next / kChunk);
            load_a(s + S - 1, buf ? buf - 1 : S - 1);
            load_b(s + S - 1, buf ? buf - 1 : S - 1);
        }
        if (wm * (BM / WM) < t.rows) compute(buf, s);  // (a wave whose rows a group's last tile has not)
        buf = buf + 1 < S ? buf + 1 : 0;
    }

    // A part's sums go to the workspace as they are.
    if (p.parts > 1) {
        float* const w = p.partial + (uint64_t)part * p.m * p.partial_stride;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const uint32_t r = wm * (BM / WM) + 16 * i + col;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const uint32_t n = n0 + wn * (BN / WN) + 16 * j + 4 * kq;
                if (r < t.rows && n < p.n) *(f32x4*)(w + (uint64_t)(t.first + r) * p.partial_stride + n) = acc[i][j];
            }
        }
        return;
    }
    // Plain outputs of 16 bits: two lanes with neighbouring column quarters exchange halves, so that each stores eight columns. (A
    // tile that ends past the last column takes the other way with all its waves: there is a barrier on it.)
    if (p.plain && NT % 2 == 0 && n0 + BN <= p.n) {
        const uint32_t nw = n0 + wn * (BN / WN);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const uint32_t r = wm * (BM / WM) + 16 * i + col;
            const bool there = r < t.rows;
            const bool none = there && p.a_rows && (uint32_t)p.a_rows[t.first + r] >= p.a_row_count;
            uint16_t* const d = (uint16_t*)p.d + (uint64_t)(t.first + r) * p.d_stride + nw + 16 * (kq & 1) + 4 * (kq & 2);
            const float scale = none ? __builtin_nanf("") : p.ab_scale;
#pragma unroll
            for (int j = 0; j < NT; j += 2) {
                uint32_t h[2][2];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        h[u][e] = fp8_pack2(p.d_dt, scale * acc[i][j + u][2 * e], scale * acc[i][j + u][2 * e + 1]);
                const auto x = __builtin_amdgcn_permlane16_swap(h[0][0], h[1][0], false, false);
                const auto y = __builtin_amdgcn_permlane16_swap(h[0][1], h[1][1], false, false);
                if (there) *(u32x4*)(d + 16 * j) = u32x4{x[0], y[0], x[1], y[1]};
            }
        }
        return;
    }
    const void* bias = p.bias ? (const uint8_t*)p.bias + t.expert * p.bias_expert * (p.d_dt == STARK_QMM_F32 ? 4 : 2) : nullptr;
    // Outputs go through LDS, a row block at a time in the wave's own part, so that whole rows are stored.
    constexpr int C = BN / WN, P = C / 4 + 1;  // columns of the wave; pieces of a row, one more than it has: rows start on other banks
    static_assert(W * 16 * P <= S * 8 * (BM + BN), "the outputs' rows fit the operands' place");
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
        const auto missing = [&](uint32_t r) { return p.a_rows && (uint32_t)p.a_rows[t.first + r] >= p.a_row_count; };
        if (p.vec) {
#pragma unroll 2
            for (int j = 0; j < NT; ++j) {
                const uint32_t row = (64 * j + lane) / (C / 4), c = (64 * j + lane) % (C / 4), r = wm * (BM / WM) + 16 * i + row;
                if (r >= t.rows) continue;
                f32x4 v = out[row * P + c];
                if (missing(r)) v = f32x4{1, 1, 1, 1} * __builtin_nanf("");
                fp8_store4(p, v, t.first + r, n0 + wn * C + 4 * c, bias);
            }
        } else {  // rows that start anywhere: a column a lane, four at a time
#pragma unroll 1
            for (int j0 = 0; j0 < 4 * NT; j0 += 4) {
                float v[4];
                uint32_t r[4], n[4];
                bool there[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    // a row is the same in every lane where it has 64 columns or more
                    const uint32_t row = C >= 64 ? (j0 + u) / (C / 64 ? C / 64 : 1) : (j0 + u) * (64 / C) + lane / C;
                    const uint32_t c = C >= 64 ? lane + 64 * ((j0 + u) % (C / 64 ? C / 64 : 1)) : lane % C;
                    r[u] = wm * (BM / WM) + 16 * i + row, n[u] = n0 + wn * C + c;
                    there[u] = r[u] < t.rows && n[u] < p.n;
                    v[u] = ((const float*)(out + row * P))[c];
                    if (there[u] && missing(r[u])) v[u] = __builtin_nanf("");
                }
                if (!p.flags) {
                    float add[4] = {0, 0, 0, 0};
                    if (bias) {
#pragma unroll
                        for (int u = 0; u < 4; ++u) add[u] = load_as_f32(bias, p.d_dt, min(n[u], p.n - 1));
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) v[u] = p.ab_scale * v[u] + add[u];
                } else {
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        if (there[u]) v[u] = fp8_finish(p, v[u], (size_t)(t.first + r[u]) * p.d_stride + n[u], bias, n[u]);
                }
                if (p.d_dt == STARK_QMM_F32) {
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        if (there[u]) ((float*)p.d + (uint64_t)(t.first + r[u]) * p.d_stride)[n[u]] = v[u];
                } else {
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        if (there[u]) ((uint16_t*)p.d + (uint64_t)(t.first + r[u]) * p.d_stride)[n[u]] = (uint16_t)fp8_pack2(p.d_dt, v[u], 0.0f);
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

template <int BM, int BN, int WM, int WN, int S, bool EXACT>
__global__ __launch_bounds__(64 * WM * WN) void fp8_tiles(Fp8Product p) {
    __shared__ TileLds<BM, BN, WM * WN, S> lds;
    const uint32_t columns = (p.n + BN - 1) / BN;
    const Fp8Groups<BM> groups(p);
    const fp8::Place at = fp8::place(fp8::tile_of(p.first_group + blockIdx.x, groups.total * columns), groups.total, columns);
    const Fp8Tile rows = groups.tile(p, at.row);
    if (rows.rows) fp8_tile<BM, BN, WM, WN, S, EXACT>(p, lds, rows, at.column * BN, blockIdx.y);
}

// The parts' sums, in their order, four columns a thread.
__global__ __launch_bounds__(256) void fp8_join(Fp8Product p) {
    const uint32_t quarters = (p.n + 3) / 4, i = blockIdx.x * 256 + threadIdx.x, row = i / quarters, n = 4 * (i % quarters);
    if (row >= p.m) return;
    const float* w = p.partial + (uint64_t)row * p.partial_stride + n;
    f32x4 v = *(const f32x4*)w;
    for (uint32_t part = 1; part < p.parts; ++part) v += *(const f32x4*)(w + (uint64_t)part * p.m * p.partial_stride);
    fp8_store4(p, v, row, n, p.bias);
}

template <int BM, int BN, int WM, int WN, int S, bool EXACT>
stark_qmm_status launch(const Fp8Product& p, hipStream_t stream) {
    const uint64_t tiles = (uint64_t)fp8::row_tiles(p.m, p.experts, BM) * ((p.n + BN - 1) / BN);
    return fp8_launch(p, (tiles + 7) / 8 * 8, 64 * WM * WN, [&](const Fp8Product& part, uint32_t groups) {
        hipLaunchKernelGGL((fp8_tiles<BM, BN, WM, WN, S, EXACT>), dim3(groups, p.parts), dim3(64 * WM * WN), 0, stream, part);
    });
}

template <bool EXACT>
stark_qmm_status launch_size(const Fp8Product& p, uint32_t tile, hipStream_t stream) {
    if (tile == 64) return launch<64, 64, 2, 2, 3, EXACT>(p, stream);
    if constexpr (!EXACT)
        if (tile == 256) return launch<256, 256, 4, 2, 2, EXACT>(p, stream);
    return launch<128, 128, 2, 2, 2, EXACT>(p, stream);
}

}  // namespace

stark_qmm_status launch_fp8_tiles(const Fp8Product& p, uint32_t tile, hipStream_t stream) {
    stark_qmm_status st = fp8_exact(p.d_dt) ? launch_size<true>(p, tile, stream) : launch_size<false>(p, tile, stream);
    if (st != STARK_QMM_OK || p.parts == 1) return st;
    hipLaunchKernelGGL(fp8_join, dim3((uint32_t)(((uint64_t)p.m * ((p.n + 3) / 4) + 255) / 256)), dim3(256), 0, stream, p);
    QMM_HIP_CHECK(hipGetLastError());
    return STARK_QMM_OK;
}

}  // namespace qmm
