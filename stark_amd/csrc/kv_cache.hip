// 4-bit paged key/value cache: the plan of a step, the append of new rows (after the rotary embedding) and the
// read of rows back. Attention over the cache: kv_attention.hip; layout: kv_layout.h.
#include "kv_common.h"

namespace {

using namespace qmm;

// ---------------------------------------------------------------- plan

constexpr uint32_t kPlanThreads = 256;
constexpr uint32_t kPlanTokens = 1024;  // tokens of a workgroup

struct PlanArgs {
    const int32_t *cached, *added, *free_pages, *free_count;
    int32_t *table, *query_start, *kv_lengths, *slots, *positions, *free_left, *status;
    uint32_t batch, capacity, free_capacity, stride, page_shift;
};

// Inclusive sum over the workgroup's 256 threads; `part` is four words of LDS.
QMM_DEVICE int64_t plan_scan(int64_t v, int64_t* part) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t u = __shfl_up((long long)v, o, 64);
        if ((int)lane >= o) v += u;
    }
    __syncthreads();  // part may still be read by the scan before
    if (lane == 63) part[wave] = v;
    __syncthreads();
    for (uint32_t w = 0; w < wave; ++w) v += part[w];
    return v;
}

// One launch, no workspace: every workgroup scans the lengths of all requests itself (256 at a time) and then
// handles 1024 of the new tokens. Each new page holds exactly one new token at its start, and that token's thread
// writes the block table's entry. Bound by latency (two dependent reads and two scans per 256 requests), not by bytes.
__global__ __launch_bounds__(kPlanThreads) void kv_plan(PlanArgs a) {
    __shared__ int64_t part[4];
    __shared__ int32_t start[kPlanThreads + 1], had[kPlanThreads], before[kPlanThreads];
    __shared__ int32_t first_page[kPlanThreads];
    __shared__ int64_t total[2];
    __shared__ uint32_t all_flags;
    const uint32_t t = threadIdx.x, n0 = blockIdx.x * kPlanTokens;
    const int32_t capacity = (int32_t)a.capacity;
    const int32_t free_count = min(max(*a.free_count, 0), (int32_t)a.free_capacity);
    const int32_t page_mask = (1 << a.page_shift) - 1;
    int64_t tokens = 0, pages = 0;  // of the requests before this pass
    uint32_t flags = 0;
    const bool first = blockIdx.x == 0;
    if (first && t == 0) a.query_start[0] = 0;
    for (uint32_t r0 = 0; r0 < a.batch; r0 += kPlanThreads) {
        const uint32_t r = r0 + t;
        const bool live = r < a.batch;
        int32_t c = live ? a.cached[r] : 0, n = live ? a.added[r] : 0;
        if (c < 0 || n < 0) flags |= STARK_QMM_KV_BAD_LENGTH;
        c = max(c, 0), n = max(n, 0);
        const int64_t end = tokens + plan_scan(n, part);
        if (end > capacity) flags |= STARK_QMM_KV_TOO_MANY_TOKENS;
        const int32_t s = (int32_t)min(end - n, (int64_t)capacity), e = (int32_t)min(end, (int64_t)capacity);
        const kv::PagePlan p = kv::page_plan(c, e - s, a.page_shift, a.stride);
        const int64_t held = (int64_t)a.stride << a.page_shift;
        if (c + (int64_t)(e - s) > held) flags |= STARK_QMM_KV_TABLE_FULL;
        const int64_t last = pages + plan_scan(p.need, part);
        if (last > free_count && p.need) flags |= STARK_QMM_KV_OUT_OF_PAGES;
        start[t] = s, had[t] = c, before[t] = p.before;
        first_page[t] = (int32_t)min(last - p.need, (int64_t)0x7fffffff);
        if (t == kPlanThreads - 1) start[kPlanThreads] = e;
        if (first && live) {
            a.query_start[r + 1] = e;
            a.kv_lengths[r] = (int32_t)min((int64_t)c + (e - s), (int64_t)0x7fffffff);
        }
        if (t == kPlanThreads - 1) total[0] = end, total[1] = last;
        __syncthreads();
        const int32_t lo = start[0], hi = start[kPlanThreads];
        for (uint32_t n = n0 + t; n < min(n0 + kPlanTokens, a.capacity); n += kPlanThreads) {
            if ((int32_t)n < lo || (int32_t)n >= hi) continue;
            uint32_t b = 0;  // last request that starts at or before n (empty ones behind it start later or hold nothing)
#pragma unroll
            for (uint32_t step = kPlanThreads / 2; step; step >>= 1)
                if (start[b + step] <= (int32_t)n) b += step;
            const int64_t pos = (int64_t)had[b] + ((int32_t)n - start[b]);
            const int64_t page = pos >> a.page_shift;
            int32_t id = -1;
            if (page < (int64_t)a.stride) {
                const size_t at = (size_t)(r0 + b) * a.stride + (size_t)page;
                if (page < before[b]) {
                    id = a.table[at];
                } else {
                    const int64_t j = first_page[b] + (page - before[b]);
                    if (j < free_count) id = a.free_pages[free_count - 1 - j];
                    if ((pos & page_mask) == 0) a.table[at] = id;
                }
            }
            const int64_t slot = id < 0 ? -1 : ((int64_t)id << a.page_shift) + (pos & page_mask);
            a.slots[n] = slot > 0x7fffffff ? -1 : (int32_t)slot;
            a.positions[n] = (int32_t)min(pos, (int64_t)0x7fffffff);
        }
        tokens = total[0], pages = total[1];
        __syncthreads();
    }
    for (uint32_t n = n0 + t; n < min(n0 + kPlanTokens, a.capacity); n += kPlanThreads)
        if ((int64_t)n >= tokens) a.slots[n] = -1, a.positions[n] = 0;
    if (!first) return;
    if (t == 0) all_flags = 0;
    __syncthreads();
    if (flags) atomicOr(&all_flags, flags);
    __syncthreads();
    if (t == 0) {
        *a.free_left = (int32_t)max((int64_t)free_count - pages, (int64_t)0);
        *a.status = (int32_t)all_flags;
    }
}

// ---------------------------------------------------------------- append

struct Rotary {
    const float2* table;
    const int32_t* positions;
    uint64_t position_stride;
    uint32_t rows, pairs, axes, interleaved;
    uint16_t axis8[16];  // the axes of eight pairs, two bits each
};

struct AppendArgs {
    KvCache cache;
    KvRows q, q_out, k, v;
    const int32_t* slots;
    uint32_t dt, tokens, heads;
    Rotary rot;
};

// Eight values of a row.
QMM_DEVICE void load8(const KvRows& r, uint32_t dt, uint32_t token, uint32_t head, uint32_t d, float* x) {
    const size_t at = (size_t)(token * r.token + head * r.head + d);
    if (r.vec) {
        if (dt == STARK_QMM_F32) {
            const float4 *p = (const float4*)((const float*)r.p + at), a = p[0], b = p[1];
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
            const u32x4 w = *(const u32x4*)((const uint16_t*)r.p + at);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t h = e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu;
                x[e] = dt == STARK_QMM_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = load_as_f32(r.p, dt, at + e);
    }
}

QMM_DEVICE void store8(const KvRows& r, uint32_t dt, uint32_t token, uint32_t head, uint32_t d, const float* x) {
    const size_t at = (size_t)(token * r.token + head * r.head + d);
    if (r.vec) {
        if (dt == STARK_QMM_F32) {
            float4* p = (float4*)((float*)r.p + at);
            p[0] = float4{x[0], x[1], x[2], x[3]}, p[1] = float4{x[4], x[5], x[6], x[7]};
        } else {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float a = x[2 * e], b = x[2 * e + 1];
                w[e] = dt == STARK_QMM_BF16 ? f32_to_bf16_bits(a) | (uint32_t)f32_to_bf16_bits(b) << 16
                                            : f32_to_f16_bits(a) | (uint32_t)f32_to_f16_bits(b) << 16;
            }
            *(u32x4*)((uint16_t*)r.p + at) = w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) store_from_f32((void*)r.p, dt, at + e, x[e]);
    }
}

// f64 to f16 through f32, two roundings, as the conversion of a 64-bit tensor does it. The barrier keeps the compiler
// from making one rounding of them.
QMM_DEVICE uint32_t f64_to_f16_bits(double v) {
    float f = (float)v;
    asm("" : "+v"(f));
    return f32_to_f16_bits(f);
}

QMM_DEVICE double shfl_xor_f64(double v, int mask) { return __shfl_xor(v, mask, 64); }

// One (token, head) row to DIM / 8 lanes of a wave, eight neighbouring values a lane: query heads first, then key
// heads, then value heads. Arithmetic in f64: a rotated value a c - b s of f32 factors has exact products and one
// rounding there, and codes, scales and biases come out as from exact arithmetic (an f32 quotient beside a half way
// point would take the wrong code, one step of the group's range / 15). Decode steps are bound by the launch.
template <int DIM>
__global__ __launch_bounds__(256) void kv_append(AppendArgs a) {
    constexpr uint32_t L = DIM / 8;  // lanes of a row
    const uint32_t heads = a.heads + 2 * a.cache.kv_heads;
    const uint64_t item = (uint64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    const uint32_t l = threadIdx.x % L, d = 8 * l;
    if (item >= (uint64_t)a.tokens * heads) return;  // whole rows: the lanes of a row leave together
    const uint32_t token = (uint32_t)(item / heads), h = (uint32_t)(item % heads);
    const bool is_q = h < a.heads, is_v = h >= a.heads + a.cache.kv_heads;
    const uint32_t head = is_q ? h : is_v ? h - a.heads - a.cache.kv_heads : h - a.heads;
    const KvRows& src = is_q ? a.q : is_v ? a.v : a.k;
    float x[8];
    load8(src, a.dt, token, head, d, x);
    double y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (double)x[e];
    const uint32_t pairs = a.rot.pairs;
    if (!is_v && d < 2 * pairs) {
        // the rotation partner's values: the same eight (interleaved), or those half the rotated width away
        const bool high = !a.rot.interleaved && d >= pairs;
        const uint32_t p0 = a.rot.interleaved ? d / 2 : high ? d - pairs : d;  // this lane's first pair
        const uint32_t np = a.rot.interleaved ? 4 : 8;
        float o[8];
        if (!a.rot.interleaved) load8(src, a.dt, token, head, high ? d - pairs : d + pairs, o);
        uint32_t axes = a.rot.axis8[p0 / 8] >> (2 * (p0 % 8));
        float2 cs[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            cs[e] = float2{0.0f, 0.0f};
            if ((uint32_t)e < np) {
                const uint32_t pos = (uint32_t)a.rot.positions[(axes & 3) * a.rot.position_stride + token];
                cs[e] = pos < a.rot.rows ? a.rot.table[(size_t)pos * pairs + p0 + e]
                                         : float2{__builtin_nanf(""), __builtin_nanf("")};
            }
            axes >>= 2;
        }
        if (a.rot.interleaved) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double u = y[2 * e], v = y[2 * e + 1], c = cs[e].x, s = cs[e].y;
                y[2 * e] = fma(u, c, -(v * s));
                y[2 * e + 1] = fma(v, c, u * s);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double c = cs[e].x, s = high ? cs[e].y : -cs[e].y;
                y[e] = fma(y[e], c, (double)o[e] * s);
            }
        }
    }
    if (is_q) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float)y[e];
        store8(a.q_out, a.dt, token, head, d, x);
        return;
    }
    // group minimum and maximum; a value that the format does not hold makes the minimum -inf
    double lo = y[0], hi = y[0];
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        lo = fmin(lo, y[e]), hi = fmax(hi, y[e]);
        bad |= !(fabs(y[e]) <= (double)kv::kLimit);
    }
    if (bad) lo = -__builtin_inf();
    const uint32_t gl = L / a.cache.groups;  // lanes of a group: 4, 8 or 16
    for (uint32_t o = 1; o < gl; o <<= 1) lo = fmin(lo, shfl_xor_f64(lo, o)), hi = fmax(hi, shfl_xor_f64(hi, o));
    bad = !(lo >= -(double)kv::kLimit);
    const uint32_t sb = bad ? 0x7e00u : f64_to_f16_bits((hi - lo) / 15.0);
    const uint32_t bb = bad ? 0x7e00u : f64_to_f16_bits(lo);
    const double s = (double)f16_bits_to_f32(sb), b = (double)f16_bits_to_f32(bb);
    uint32_t w = 0;
    if (s > 0.0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w |= (uint32_t)fmin(fmax(rint((y[e] - b) / s), 0.0), 15.0) << (4 * e);
    }
    const uint32_t slot = (uint32_t)a.slots[token];
    const uint32_t page = slot >> a.cache.page_shift, page_size = 1u << a.cache.page_shift;
    const bool stored = page < a.cache.page_count;
    const uint32_t in_page = slot & (page_size - 1), t = in_page % kv::kTile;
    uint8_t* rec = a.cache.data + kv::record_index(stored ? page : 0, a.cache.kv_heads, head, page_size, in_page) *
                                      (uint64_t)a.cache.record;
    const uint32_t half_rec = kv::codes_bytes(DIM) + kv::planes_bytes(a.cache.groups);
    if (is_v) rec += half_rec;
    if (stored && l % gl == 0)
        *(uint32_t*)(rec + kv::codes_bytes(DIM) + kv::plane_word(t, l / gl)) = sb | bb << 16;
    if (!is_v) {
        if (stored) *(uint32_t*)(rec + kv::key_word(DIM, t, l)) = w;
        return;
    }
    // value bytes: byte i of lane r is byte r % 4 of code word 4 i + r / 4 (of its half of the head)
    const int row = (int)(threadIdx.x & 63) - (int)l;
    if (DIM == 64) {
#pragma unroll
        for (uint32_t j = 0; j < 2; ++j) {
            const uint32_t r = 2 * l + j;
            uint32_t out = 0;
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i)
                out |= ((uint32_t)__shfl((int)w, row + (int)(4 * i + r / 4), 64) >> (8 * (r % 4)) & 0xffu) << (8 * i);
            if (stored) *(uint16_t*)(rec + kv::value_byte(DIM, t, 0, r, 0)) = (uint16_t)out;
        }
    } else {
        const uint32_t r = l % 16, half = l / 16;
        uint32_t out = 0;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            out |= ((uint32_t)__shfl((int)w, row + (int)(16 * half + 4 * i + r / 4), 64) >> (8 * (r % 4)) & 0xffu)
                   << (8 * i);
        if (stored) *(uint32_t*)(rec + kv::value_byte(DIM, t, half, r, 0)) = out;
    }
}

// ---------------------------------------------------------------- read

struct ReadArgs {
    KvCache cache;
    KvRows k, v;
    const int32_t* slots;
    uint32_t dt, tokens;
};

// Eight neighbouring values to a lane, as in kv_append. s * code + b: the product of an f16 scale and a code is
// exact in f32, so each value is rounded once (twice to 16 bits). Bound by HBM writes.
template <int DIM>
__global__ __launch_bounds__(256) void kv_read(ReadArgs a) {
    constexpr uint32_t L = DIM / 8;
    const uint32_t heads = 2 * a.cache.kv_heads;
    const uint64_t item = (uint64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    const uint32_t l = threadIdx.x % L;
    if (item >= (uint64_t)a.tokens * heads) return;
    const uint32_t token = (uint32_t)(item / heads), h = (uint32_t)(item % heads);
    const bool is_v = h >= a.cache.kv_heads;
    const uint32_t head = is_v ? h - a.cache.kv_heads : h;
    const KvRows& dst = is_v ? a.v : a.k;
    const uint32_t slot = (uint32_t)a.slots[token];
    const uint32_t page = slot >> a.cache.page_shift, page_size = 1u << a.cache.page_shift;
    if (!dst.p || page >= a.cache.page_count) return;
    const uint32_t in_page = slot & (page_size - 1), t = in_page % kv::kTile;
    const uint8_t* rec = a.cache.data + kv::record_index(page, a.cache.kv_heads, head, page_size, in_page) *
                                            (uint64_t)a.cache.record;
    if (is_v) rec += kv::codes_bytes(DIM) + kv::planes_bytes(a.cache.groups);
    const uint32_t plane = *(const uint32_t*)(rec + kv::codes_bytes(DIM) + kv::plane_word(t, l * a.cache.groups / L));
    const float s = f16_bits_to_f32(plane & 0xffffu), b = f16_bits_to_f32(plane >> 16);
    uint32_t w = 0;
    if (!is_v) {
        w = *(const uint32_t*)(rec + kv::key_word(DIM, t, l));
    } else {
        const uint32_t half = l / 16, i = l % 16 / 4;
#pragma unroll
        for (uint32_t m = 0; m < 4; ++m)
            w |= (uint32_t)rec[kv::value_byte(DIM, t, half, 4 * (l % 4) + m, i)] << (8 * m);
    }
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf(s, (float)(w >> (4 * e) & 15u), b);
    store8(dst, a.dt, token, head, 8 * l, x);
}

// Rows of DIM / 8 lanes, 256 lanes a workgroup; the grid stays below 2^24 workgroups.
template <class F>
stark_qmm_status launch_rows(uint32_t dim, uint64_t rows, F launch) {
    if (rows == 0) return STARK_QMM_OK;
    const uint64_t per = 256 / (dim / 8), blocks = (rows + per - 1) / per;
    if (blocks >= 1ull << 24) return STARK_QMM_UNSUPPORTED;
    launch(dim3((uint32_t)blocks));
    QMM_HIP_CHECK(hipGetLastError());
    return STARK_QMM_OK;
}

bool dt_ok(uint32_t dt) { return dt == STARK_QMM_F32 || dt == STARK_QMM_F16 || dt == STARK_QMM_BF16; }

}  // namespace

extern "C" {

stark_qmm_status stark_qmm_kv_cache_size(const stark_qmm_kv_cache* cache, uint64_t* bytes) {
    if (!cache || !bytes) return STARK_QMM_INVALID_ARGUMENT;
    KvCache c;
    return kv_geometry(*cache, &c, bytes);
}

stark_qmm_status stark_qmm_kv_plan(const stark_qmm_kv_plan_args* p, void* stream) {
    if (!p) return STARK_QMM_INVALID_ARGUMENT;
    if (p->struct_size != sizeof(*p)) return STARK_QMM_ABI_MISMATCH;
    if (p->page_size < 16 || p->page_size > 1024 || (p->page_size & (p->page_size - 1))) return STARK_QMM_INVALID_ARGUMENT;
    if (p->batch > (1u << 20) || p->token_capacity > (1u << 24) || p->free_capacity > 0x7fffffffu)
        return STARK_QMM_INVALID_ARGUMENT;
    if ((uint64_t)p->table_stride * p->page_size > 0x7fffffffull) return STARK_QMM_INVALID_ARGUMENT;
    if (!p->free_count || !p->query_start || !p->free_left || !p->status) return STARK_QMM_INVALID_ARGUMENT;
    if (p->batch && (!p->cached || !p->added || !p->kv_lengths || (p->table_stride && !p->block_table)))
        return STARK_QMM_INVALID_ARGUMENT;
    if ((p->token_capacity && (!p->slots || !p->positions)) || (p->free_capacity && !p->free_pages))
        return STARK_QMM_INVALID_ARGUMENT;
    const void* all[] = {p->cached, p->added, p->free_pages, p->free_count, p->block_table, p->query_start, p->kv_lengths,
                         p->slots, p->positions, p->free_left, p->status};
    for (const void* x : all)
        if (!kv_aligned(x, 4)) return STARK_QMM_INVALID_ARGUMENT;
    PlanArgs a{p->cached, p->added, p->free_pages, p->free_count, p->block_table, p->query_start, p->kv_lengths, p->slots,
               p->positions, p->free_left, p->status, p->batch, p->token_capacity, p->free_capacity, p->table_stride, 4};
    while ((1u << a.page_shift) < p->page_size) ++a.page_shift;
    const uint32_t blocks = std::max(1u, (p->token_capacity + kPlanTokens - 1) / kPlanTokens);
    hipLaunchKernelGGL(kv_plan, dim3(blocks), dim3(kPlanThreads), 0, (hipStream_t)stream, a);
    QMM_HIP_CHECK(hipGetLastError());
    return STARK_QMM_OK;
}

stark_qmm_status stark_qmm_kv_append(const stark_qmm_kv_append_args* p, void* stream) {
    if (!p) return STARK_QMM_INVALID_ARGUMENT;
    if (p->struct_size != sizeof(*p)) return STARK_QMM_ABI_MISMATCH;
    AppendArgs a{};
    const stark_qmm_status st = kv_view(p->cache, &a.cache);
    if (st != STARK_QMM_OK) return st;
    if (!dt_ok(p->data_type)) return STARK_QMM_UNSUPPORTED_DATA_TYPE;
    const uint32_t dim = a.cache.dim, heads = p->q ? p->heads : 0, dt = p->data_type;
    if ((p->q == nullptr) != (p->q_out == nullptr) || (p->q && (p->heads == 0 || p->heads > 65536)))
        return STARK_QMM_INVALID_ARGUMENT;
    if (p->tokens > (1u << 24)) return STARK_QMM_INVALID_ARGUMENT;
    if (p->tokens == 0) return STARK_QMM_OK;
    if (!p->slots || !kv_aligned(p->slots, 4)) return STARK_QMM_INVALID_ARGUMENT;
    if (!kv_rows_ok(p->k, p->k_token_stride, p->k_head_stride, p->tokens, a.cache.kv_heads, dim, dt) ||
        !kv_rows_ok(p->v, p->v_token_stride, p->v_head_stride, p->tokens, a.cache.kv_heads, dim, dt))
        return STARK_QMM_INVALID_ARGUMENT;
    if (p->q && (!kv_rows_ok(p->q, p->q_token_stride, p->q_head_stride, p->tokens, heads, dim, dt) ||
                 !kv_rows_ok(p->q_out, p->q_out_token_stride, p->q_out_head_stride, p->tokens, heads, dim, dt)))
        return STARK_QMM_INVALID_ARGUMENT;
    const stark_qmm_rotary& r = p->rotary;
    if (r.rotary_dim) {
        if (r.rotary_dim % 16 || r.rotary_dim > dim || r.axes < 1 || r.axes > 4) return STARK_QMM_INVALID_ARGUMENT;
        if (!r.table || !kv_aligned(r.table, 8) || !r.positions || !kv_aligned(r.positions, 4) ||
            r.table_rows > 0x7fffffffu || (r.axes > 1 && (r.position_stride < p->tokens || r.position_stride >> 32)))
            return STARK_QMM_INVALID_ARGUMENT;
        a.rot = Rotary{(const float2*)r.table, r.positions, r.axes > 1 ? r.position_stride : 0, r.table_rows,
                       r.rotary_dim / 2, r.axes, r.interleaved != 0, {}};
        for (uint32_t i = 0; i < a.rot.pairs; ++i) {
            if (r.axis_of_pair[i] >= r.axes) return STARK_QMM_INVALID_ARGUMENT;
            a.rot.axis8[i / 8] |= (uint16_t)(r.axis_of_pair[i] << (2 * (i % 8)));
        }
    }
    a.q = kv_rows(p->q, p->q_token_stride, p->q_head_stride, dt);
    a.q_out = kv_rows(p->q_out, p->q_out_token_stride, p->q_out_head_stride, dt);
    a.k = kv_rows(p->k, p->k_token_stride, p->k_head_stride, dt);
    a.v = kv_rows(p->v, p->v_token_stride, p->v_head_stride, dt);
    a.slots = p->slots;
    a.dt = dt, a.tokens = p->tokens, a.heads = heads;
    const hipStream_t s = (hipStream_t)stream;
    return launch_rows(dim, (uint64_t)p->tokens * (heads + 2 * a.cache.kv_heads), [&](dim3 grid) {
        if (dim == 64) hipLaunchKernelGGL(kv_append<64>, grid, dim3(256), 0, s, a);
        else if (dim == 128) hipLaunchKernelGGL(kv_append<128>, grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL(kv_append<256>, grid, dim3(256), 0, s, a);
    });
}

stark_qmm_status stark_qmm_kv_read(const stark_qmm_kv_read_args* p, void* stream) {
    if (!p) return STARK_QMM_INVALID_ARGUMENT;
    if (p->struct_size != sizeof(*p)) return STARK_QMM_ABI_MISMATCH;
    ReadArgs a{};
    const stark_qmm_status st = kv_view(p->cache, &a.cache);
    if (st != STARK_QMM_OK) return st;
    if (!dt_ok(p->data_type)) return STARK_QMM_UNSUPPORTED_DATA_TYPE;
    if (p->tokens > (1u << 24) || (!p->k && !p->v)) return STARK_QMM_INVALID_ARGUMENT;
    if (p->tokens == 0) return STARK_QMM_OK;
    if (!p->slots || !kv_aligned(p->slots, 4)) return STARK_QMM_INVALID_ARGUMENT;
    const uint32_t dim = a.cache.dim, dt = p->data_type;
    if ((p->k && !kv_rows_ok(p->k, p->k_token_stride, p->k_head_stride, p->tokens, a.cache.kv_heads, dim, dt)) ||
        (p->v && !kv_rows_ok(p->v, p->v_token_stride, p->v_head_stride, p->tokens, a.cache.kv_heads, dim, dt)))
        return STARK_QMM_INVALID_ARGUMENT;
    a.k = kv_rows(p->k, p->k_token_stride, p->k_head_stride, dt);
    a.v = kv_rows(p->v, p->v_token_stride, p->v_head_stride, dt);
    a.slots = p->slots;
    a.dt = dt, a.tokens = p->tokens;
    const hipStream_t s = (hipStream_t)stream;
    return launch_rows(dim, (uint64_t)p->tokens * 2 * a.cache.kv_heads, [&](dim3 grid) {
        if (dim == 64) hipLaunchKernelGGL(kv_read<64>, grid, dim3(256), 0, s, a);
        else if (dim == 128) hipLaunchKernelGGL(kv_read<128>, grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL(kv_read<256>, grid, dim3(256), 0, s, a);
    });
}

}  // extern "C"
