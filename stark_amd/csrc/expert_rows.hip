// Routes of a step's experts in expert order, and the weighted sum of each token's expert rows.
#include "fp8_common.h"

namespace qmm {
namespace {

// ---- plan: a stable counting sort of the routes by expert.
//
// A wave ranks 64 consecutive routes at a time: lanes with the same expert find each other by one ballot for each bit of the
// id, a lane's rank is the wave's count of that expert so far and the lower lanes among them. So positions do not depend on
// the order in which anything runs. A workgroup's sixteen waves take consecutive runs of its routes; a call of more than one
// workgroup counts first (plan_count), and each workgroup adds up what the ones before it have (plan_place).
// Latency bounds it, so a wave has as few turns as 256 workgroups allow.
constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr uint32_t kMaxExperts = 1024;
// Routes that one workgroup takes without counting first (2048 routes 5.8 us, with a count 7.4; 4096 routes 8.9 and 7.6; 65536
// routes 17.6 us with 4096 to a workgroup, 10.0 with 1024).
constexpr uint32_t kOneGroup = 2048;

struct Plan {
    const uint32_t* ids;
    int32_t* group_start;
    int32_t* tokens;
    int32_t* slots;
    uint32_t* counts;  // [workgroups, experts]
    uint32_t routes, active, experts, first, groups, per_group, bits;
};

// Lanes of the wave whose key is this lane's.
QMM_DEVICE uint64_t same_key(uint32_t key, uint32_t bits) {
    uint64_t m = ~0ull;
    for (uint32_t b = 0; b < bits; ++b) {
        const uint64_t set = __ballot((key >> b) & 1);
        m &= (key >> b) & 1 ? set : ~set;
    }
    return m;
}

// Key of a route: its expert here, or `experts`.
QMM_DEVICE uint32_t route_key(const Plan& p, uint32_t r, uint32_t end) {
    if (r >= end) return p.experts;
    const uint32_t e = p.ids[r] - p.first;
    return min(e, p.experts);
}

// Routes of this wave: [begin, end), whole 64s but the last.
QMM_DEVICE void wave_routes(const Plan& p, uint32_t wave, uint32_t* begin, uint32_t* end) {
    const uint32_t g0 = blockIdx.x * p.per_group, g1 = min(g0 + p.per_group, p.routes);
    const uint32_t per_wave = (p.per_group / 64 + kPlanWaves - 1) / kPlanWaves * 64;
    *begin = min(g0 + wave * per_wave, g1);
    *end = min(*begin + per_wave, g1);
}

// The wave's routes of each expert into cnt[], which holds what came before them; `place` gets route, key and rank.
template <typename F>
QMM_DEVICE void rank_routes(const Plan& p, uint32_t begin, uint32_t end, uint32_t* cnt, const F& place) {
    const uint32_t lane = threadIdx.x & 63;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (uint32_t r0 = begin; r0 < end; r0 += 64) {
        const uint32_t r = r0 + lane, key = route_key(p, r, end);
        const uint64_t same = same_key(key, p.bits);
        const uint32_t below = __popcll(same & ((1ull << lane) - 1));
        const uint32_t before = key < p.experts ? cnt[key] : 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (key < p.experts && below == 0) cnt[key] = before + __popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (r < end) place(r, key, before + below);
    }
}

__global__ __launch_bounds__(kPlanThreads) void plan_count(Plan p) {
    __shared__ uint32_t cnt[kPlanWaves][kMaxExperts];
    const uint32_t tid = threadIdx.x, wave = tid >> 6;
    for (uint32_t e = tid & 63; e < p.experts; e += 64) cnt[wave][e] = 0;
    uint32_t begin, end;
    wave_routes(p, wave, &begin, &end);
    rank_routes(p, begin, end, cnt[wave], [](uint32_t, uint32_t, uint32_t) {});
    __syncthreads();
    for (uint32_t e = tid; e < p.experts; e += kPlanThreads) {
        uint32_t n = 0;
        for (int w = 0; w < kPlanWaves; ++w) n += cnt[w][e];
        p.counts[(size_t)blockIdx.x * p.experts + e] = n;
    }
}

__global__ __launch_bounds__(kPlanThreads) void plan_place(Plan p) {
    __shared__ uint32_t cnt[kPlanWaves][kMaxExperts];
    __shared__ uint32_t sums[kPlanWaves], part[2][kPlanThreads];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (uint32_t e = lane; e < p.experts; e += 64) cnt[wave][e] = 0;
    uint32_t begin, end;
    wave_routes(p, wave, &begin, &end);
    rank_routes(p, begin, end, cnt[wave], [](uint32_t, uint32_t, uint32_t) {});
    __syncthreads();
    // thread e: the routes of expert e in all, before this workgroup, and in its waves
    uint32_t before = 0, all = 0;
    if (p.groups > 1) {
        // slices of the threads take every so many groups' counts, all loads in flight
        const uint32_t wide = (p.experts + 63) / 64 * 64, slices = kPlanThreads / wide, slice = tid / wide, e = tid % wide;
        if (slice < slices && e < p.experts) {
#pragma unroll 8
            for (uint32_t g = slice; g < p.groups; g += slices) {
                const uint32_t n = p.counts[(size_t)g * p.experts + e];
                all += n;
                before += g < blockIdx.x ? n : 0;
            }
        }
        part[0][tid] = all, part[1][tid] = before;
        __syncthreads();
        all = before = 0;
        if (tid < p.experts)
            for (uint32_t i = 0; i < slices; ++i) all += part[0][i * wide + tid], before += part[1][i * wide + tid];
    } else if (tid < p.experts) {
        for (int w = 0; w < kPlanWaves; ++w) all += cnt[w][tid];
    }
    uint32_t start = all;  // inclusive scan over the experts
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t u = __shfl_up(start, d, 64);
        if (lane >= (uint32_t)d) start += u;
    }
    if (lane == 63) sums[wave] = start;
    __syncthreads();
    uint32_t total = 0;
    for (uint32_t w = 0; w < kPlanWaves; ++w) {
        start += w < wave ? sums[w] : 0;
        total += sums[w];
    }
    start -= all;
    if (tid < p.experts) {
        uint32_t at = start + before;
        for (int w = 0; w < kPlanWaves; ++w) {
            const uint32_t n = cnt[w][tid];
            cnt[w][tid] = at;
            at += n;
        }
        if (blockIdx.x == 0) {
            p.group_start[tid] = (int32_t)start;
            if (tid == 0) p.group_start[p.experts] = (int32_t)total;
        }
    }
    __syncthreads();
    rank_routes(p, begin, end, cnt[wave], [&](uint32_t r, uint32_t key, uint32_t rank) {
        const bool here = key < p.experts;
        p.slots[r] = here ? (int32_t)rank : -1;
        if (here) p.tokens[rank] = (int32_t)(r / p.active);
        if (r >= total) p.tokens[r] = -1;  // positions behind the last
    });
}

// Routes of a workgroup: whole turns of its waves, and at most 256 workgroups.
uint32_t plan_routes(uint32_t routes) { return routes <= kOneGroup ? (routes + 63) / 64 * 64 : std::max(1u, (routes + 262143) / 262144) * 1024; }
uint32_t plan_groups(uint32_t routes) { return routes <= kOneGroup ? 1 : (routes + plan_routes(routes) - 1) / plan_routes(routes); }

stark_qmm_status check_plan(const stark_qmm_expert_plan_args* a, uint64_t* bytes) {
    if (!a || !bytes) return STARK_QMM_INVALID_ARGUMENT;
    if (a->struct_size != sizeof(*a)) return STARK_QMM_ABI_MISMATCH;
    if (a->experts == 0 || a->experts > kMaxExperts || a->active == 0 || (uint64_t)a->tokens * a->active > (1u << 24))
        return STARK_QMM_INVALID_ARGUMENT;
    const uint32_t groups = plan_groups(a->tokens * a->active);
    *bytes = groups > 1 ? (4ull * groups * a->experts + 15) / 16 * 16 : 0;
    return STARK_QMM_OK;
}

// ---- combine: a workgroup takes a token and 2048 values of its row (1024 in f32, or where rows start anywhere). A thread has 16
// bytes of a row, or four values 256 apart; the rows of four routes are loaded together. HBM bounds it.
constexpr int kSumThreads = 256, kSumRoutes = 4;

struct Combine {
    const void* x;
    const int32_t* slots;
    const float* weights;
    void* out;
    uint64_t x_stride, out_stride;
    uint32_t active, rows, width, accumulate;
};

template <uint32_t DT, bool VEC>
struct SumValues {
    static constexpr int kCount = VEC && DT != STARK_QMM_F32 ? 8 : 4;
    float v[kCount];
    // values of a row from column c on
    QMM_DEVICE void load(const void* p, size_t row, uint32_t c, uint32_t width) {
        if constexpr (!VEC) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = load_as_f32(p, DT, row + min(c + e * kSumThreads, width - 1));
        } else if constexpr (DT == STARK_QMM_F32) {
            const f32x4 t = *(const f32x4*)((const float*)p + row + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = t[e];
        } else {
            const u32x4 t = *(const u32x4*)((const uint16_t*)p + row + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[2 * e] = DT == STARK_QMM_BF16 ? __uint_as_float(t[e] << 16) : f16_bits_to_f32(t[e] & 0xffffu);
                v[2 * e + 1] = DT == STARK_QMM_BF16 ? __uint_as_float(t[e] & 0xffff0000u) : f16_bits_to_f32(t[e] >> 16);
            }
        }
    }
    QMM_DEVICE void store(void* p, size_t row, uint32_t c, uint32_t width) const {
        if constexpr (!VEC) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e * kSumThreads < width) store_from_f32(p, DT, row + c + e * kSumThreads, v[e]);
        } else if constexpr (DT == STARK_QMM_F32) {
            *(f32x4*)((float*)p + row + c) = f32x4{v[0], v[1], v[2], v[3]};
        } else {
            u32x4 t;
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = fp8_pack2(DT, v[2 * e], v[2 * e + 1]);
            *(u32x4*)((uint16_t*)p + row + c) = t;
        }
    }
};

template <uint32_t DT, bool VEC>
__global__ __launch_bounds__(kSumThreads) void expert_combine(Combine q) {
    using Values = SumValues<DT, VEC>;
    constexpr int E = Values::kCount;
    const uint32_t token = blockIdx.x, c = blockIdx.y * kSumThreads * E + threadIdx.x * (VEC ? E : 1);
    if (c >= q.width) return;
    Values sum;
#pragma unroll
    for (int e = 0; e < E; ++e) sum.v[e] = 0.0f;
    const size_t out = (size_t)token * q.out_stride, route = (size_t)token * q.active;
    if (q.accumulate) sum.load(q.out, out, c, q.width);
    for (uint32_t j = 0; j < q.active; j += kSumRoutes) {
        uint32_t slot[kSumRoutes];
        float w[kSumRoutes];
        Values x[kSumRoutes];
#pragma unroll
        for (int u = 0; u < kSumRoutes; ++u) {
            const size_t at = route + min(j + u, q.active - 1);
            slot[u] = j + u < q.active ? (uint32_t)q.slots[at] : q.rows;
            w[u] = q.weights[at];
        }
#pragma unroll
        for (int u = 0; u < kSumRoutes; ++u)
            if (slot[u] < q.rows) x[u].load(q.x, (size_t)slot[u] * q.x_stride, c, q.width);
#pragma unroll
        for (int u = 0; u < kSumRoutes; ++u)
            if (slot[u] < q.rows) {
#pragma unroll
                for (int e = 0; e < E; ++e) sum.v[e] = fmaf(w[u], x[u].v[e], sum.v[e]);
            }
    }
    sum.store(q.out, out, c, q.width);
}

template <uint32_t DT>
void launch_combine(const Combine& q, uint32_t tokens, bool vec, hipStream_t s) {
    const uint32_t each = kSumThreads * (vec && DT != STARK_QMM_F32 ? 8 : 4);
    const dim3 grid(tokens, (q.width + each - 1) / each);
    if (vec) hipLaunchKernelGGL((expert_combine<DT, true>), grid, dim3(kSumThreads), 0, s, q);
    else hipLaunchKernelGGL((expert_combine<DT, false>), grid, dim3(kSumThreads), 0, s, q);
}

}  // namespace
}  // namespace qmm

extern "C" {

stark_qmm_status stark_qmm_expert_plan_workspace_size(const stark_qmm_expert_plan_args* args, uint64_t* bytes) {
    return qmm::check_plan(args, bytes);
}

stark_qmm_status stark_qmm_expert_plan(const stark_qmm_expert_plan_args* a, void* stream) {
    using namespace qmm;
    uint64_t need = 0;
    const stark_qmm_status st = check_plan(a, &need);
    if (st != STARK_QMM_OK) return st;
    const uint32_t routes = a->tokens * a->active;
    if (!a->group_start || (routes && (!a->ids || !a->tokens_out || !a->slots))) return STARK_QMM_INVALID_ARGUMENT;
    if (!fp8_aligned(a->ids, 4) || !fp8_aligned(a->group_start, 4) || !fp8_aligned(a->tokens_out, 4) || !fp8_aligned(a->slots, 4))
        return STARK_QMM_INVALID_ARGUMENT;
    const uint64_t rn = 4ull * routes, gn = 4ull * (a->experts + 1);
    const void* ranges[] = {a->ids, a->tokens_out, a->slots, a->group_start, a->workspace};
    const uint64_t sizes[] = {rn, rn, rn, gn, need};
    for (int i = 0; i < 5; ++i)
        for (int j = 0; j < i; ++j)
            if (fp8_overlap(ranges[i], sizes[i], ranges[j], sizes[j])) return STARK_QMM_INVALID_ARGUMENT;
    if (need && (!a->workspace || !fp8_aligned(a->workspace, 16))) return STARK_QMM_INVALID_ARGUMENT;
    if (need > a->workspace_size) return STARK_QMM_WORKSPACE_TOO_SMALL;
    Plan p{a->ids, a->group_start, a->tokens_out, a->slots, (uint32_t*)a->workspace, routes, a->active, a->experts, a->first,
           plan_groups(routes), plan_routes(routes), 0};
    while ((1u << p.bits) <= a->experts) ++p.bits;  // keys are 0 .. experts
    if (p.groups > 1) {
        hipLaunchKernelGGL(plan_count, dim3(p.groups), dim3(kPlanThreads), 0, (hipStream_t)stream, p);
        QMM_HIP_CHECK(hipGetLastError());
    }
    hipLaunchKernelGGL(plan_place, dim3(p.groups), dim3(kPlanThreads), 0, (hipStream_t)stream, p);
    QMM_HIP_CHECK(hipGetLastError());
    return STARK_QMM_OK;
}

stark_qmm_status stark_qmm_expert_combine(const stark_qmm_expert_combine_args* a, void* stream) {
    using namespace qmm;
    if (!a) return STARK_QMM_INVALID_ARGUMENT;
    if (a->struct_size != sizeof(*a)) return STARK_QMM_ABI_MISMATCH;
    if (!fp8_type(a->data_type)) return STARK_QMM_UNSUPPORTED_DATA_TYPE;
    if (a->active == 0 || a->active > 1024 || a->tokens >= (1u << 24) || a->width > (1u << 24) || a->rows > 0x7fffffffu)
        return STARK_QMM_INVALID_ARGUMENT;
    if (a->tokens == 0 || a->width == 0) return STARK_QMM_OK;
    const uint64_t e = fp8_element(a->data_type), routes = (uint64_t)a->tokens * a->active;
    if (!a->slots || !a->weights || !a->out || (a->rows && !a->x)) return STARK_QMM_INVALID_ARGUMENT;
    if (!fp8_aligned(a->x, e) || !fp8_aligned(a->out, e) || !fp8_aligned(a->slots, 4) || !fp8_aligned(a->weights, 4))
        return STARK_QMM_INVALID_ARGUMENT;
    if ((a->x_row_stride | a->out_row_stride) >> 40) return STARK_QMM_INVALID_ARGUMENT;
    if ((a->rows > 1 && a->x_row_stride < a->width) || (a->tokens > 1 && a->out_row_stride < a->width)) return STARK_QMM_INVALID_ARGUMENT;
    const uint64_t xs = a->rows > 1 ? a->x_row_stride : 0, os = a->tokens > 1 ? a->out_row_stride : 0;
    const uint64_t on = e * fp8_span(a->tokens, os, a->width);
    if (fp8_overlap(a->out, on, a->x, e * fp8_span(a->rows, xs, a->width)) || fp8_overlap(a->out, on, a->slots, 4 * routes) ||
        fp8_overlap(a->out, on, a->weights, 4 * routes))
        return STARK_QMM_INVALID_ARGUMENT;
    const Combine q{a->x, a->slots, a->weights, a->out, xs, os, a->active, a->rows, a->width, a->accumulate};
    const uint64_t unit = 16 / e;
    const bool vec = fp8_aligned(a->x, 16) && fp8_aligned(a->out, 16) && xs % unit == 0 && os % unit == 0 && a->width % unit == 0;
    if (a->data_type == STARK_QMM_F32) launch_combine<STARK_QMM_F32>(q, a->tokens, vec, (hipStream_t)stream);
    else if (a->data_type == STARK_QMM_F16) launch_combine<STARK_QMM_F16>(q, a->tokens, vec, (hipStream_t)stream);
    else launch_combine<STARK_QMM_BF16>(q, a->tokens, vec, (hipStream_t)stream);
    QMM_HIP_CHECK(hipGetLastError());
    return STARK_QMM_OK;
}

}  // extern "C"
