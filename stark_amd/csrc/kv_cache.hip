// 4-bit paged key/value cache: the plan of a step, the append of new rows (after the rotary embedding) and the
// read of rows back. Attention over the cache: kv_attention.hip; layout: kv_layout.h.
#include <type_traits>

#include "kv_common.h"

namespace {

using namespace qmm;

// ---------------------------------------------------------------- plan

constexpr uint32_t kPlanThreads = 256;

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

// One launch, no workspace: every workgroup scans the lengths of all requests itself (256 N at a time, N neighbours to a
// thread) and then handles 256 of the new tokens. Each new page holds exactly one new token at its start, and that token's
// thread writes the block table's entry. Bound by latency (two dependent reads and two scans a pass, then a table entry's
// read), not by bytes: 3.3 us for 8 requests of one token, 4.7 for 512 with 24 chunks, 11.4 for 4096. With one request a
// thread 5.5 and 25 (but 4.2 against 4.5 for 256), with 1024 tokens a workgroup 7.0 and 14.7.
template <int N>
__global__ __launch_bounds__(kPlanThreads) void kv_plan(PlanArgs a) {
    constexpr uint32_t kPass = kPlanThreads * N;  // requests
    __shared__ int64_t part[4];
    __shared__ int32_t start[kPass + 1], had[kPass], before[kPass];
    __shared__ int32_t first_page[kPass];
    __shared__ int64_t total[2];
    __shared__ uint32_t all_flags;
    const uint32_t t = threadIdx.x, token = blockIdx.x * kPlanThreads + t;
    const int32_t capacity = (int32_t)a.capacity;
    const int32_t free_count = min(max(*a.free_count, 0), (int32_t)a.free_capacity);
    const int32_t page_mask = (1 << a.page_shift) - 1;
    int64_t tokens = 0, pages = 0;  // of the requests before this pass
    uint32_t flags = 0;
    const bool first = blockIdx.x == 0;
    if (first && t == 0) a.query_start[0] = 0;
    for (uint32_t r0 = 0; r0 < a.batch; r0 += kPass) {
        const uint32_t r = r0 + t * N;
        int32_t c[N], n[N];
        int64_t added = 0, need = 0;  // of the thread's requests
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool live = r + i < a.batch;
            c[i] = live ? a.cached[r + i] : 0, n[i] = live ? a.added[r + i] : 0;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (c[i] < 0 || n[i] < 0) flags |= STARK_QMM_KV_BAD_LENGTH;
            c[i] = max(c[i], 0), n[i] = max(n[i], 0);
            added += n[i];
        }
        int64_t end = tokens + plan_scan(added, part) - added;
        int32_t s[N], e[N], need_i[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s[i] = (int32_t)min(end, (int64_t)capacity);
            end += n[i];
            if (end > capacity && n[i]) flags |= STARK_QMM_KV_TOO_MANY_TOKENS;
            e[i] = (int32_t)min(end, (int64_t)capacity);
            const kv::PagePlan p = kv::page_plan(c[i], e[i] - s[i], a.page_shift, a.stride);
            const int64_t held = (int64_t)a.stride << a.page_shift;
            if (c[i] + (int64_t)(e[i] - s[i]) > held) flags |= STARK_QMM_KV_TABLE_FULL;
            need_i[i] = p.need, need += p.need;
            start[t * N + i] = s[i], had[t * N + i] = c[i], before[t * N + i] = p.before;
        }
        int64_t last = pages + plan_scan(need, part) - need;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            first_page[t * N + i] = (int32_t)min(last, (int64_t)0x7fffffff);
            last += need_i[i];
            if (last > free_count && need_i[i]) flags |= STARK_QMM_KV_OUT_OF_PAGES;
            if (first && r + i < a.batch) {
                a.query_start[r + i + 1] = e[i];
                a.kv_lengths[r + i] = (int32_t)min((int64_t)c[i] + (e[i] - s[i]), (int64_t)0x7fffffff);
            }
        }
        if (t == kPlanThreads - 1) start[kPass] = e[N - 1], total[0] = end, total[1] = last;
        __syncthreads();
        const int32_t lo = start[0], hi = start[kPass];
        if (token < a.capacity && (int32_t)token >= lo && (int32_t)token < hi) {
            uint32_t b = 0;  // last request that starts at or before it (empty ones behind it start later or hold nothing)
#pragma unroll
            for (uint32_t step = kPass / 2; step; step >>= 1)
                if (start[b + step] <= (int32_t)token) b += step;
            const int64_t pos = (int64_t)had[b] + ((int32_t)token - start[b]);
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
            a.slots[token] = slot > 0x7fffffff ? -1 : (int32_t)slot;
            a.positions[token] = (int32_t)min(pos, (int64_t)0x7fffffff);
        }
        tokens = total[0], pages = total[1];
        __syncthreads();
    }
    if (token < a.capacity && (int64_t)token >= tokens) a.slots[token] = -1, a.positions[token] = 0;
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
    uint32_t one_axis;    // the eight pairs of each octet turn by one axis, and rows of the table are 16-byte aligned
    uint16_t axis8[16];   // the axes of eight pairs, two bits each
};

struct AppendArgs {
    KvCache cache;
    KvRows q, q_out, k, v;
    const int32_t* slots;
    uint32_t tokens, heads;
    uint32_t sets;  // threads of a lane place that share a token's heads: set i takes heads i, i + sets, ...
    Rotary rot;
};

// Eight neighbouring values of a row as they are stored. Rows of any alignment: the compiler makes one unaligned 16-byte
// access of the elements.
template <uint32_t DT>
struct Eight {
    static constexpr int kWords = DT == STARK_QMM_F32 ? 8 : 4;
    uint32_t w[kWords];

    QMM_DEVICE void load(const KvRows& r, uint32_t token, uint32_t head, uint32_t d) {
        const size_t at = (size_t)(token * r.token + head * r.head + d);
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if (DT == STARK_QMM_F32) w[i] = ((const uint32_t*)r.p)[at + i];
            else w[i] = ((const uint16_t*)r.p)[at + 2 * i] | (uint32_t)((const uint16_t*)r.p)[at + 2 * i + 1] << 16;
        }
    }
    QMM_DEVICE void store(const KvRows& r, uint32_t token, uint32_t head, uint32_t d) const {
        const size_t at = (size_t)(token * r.token + head * r.head + d);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (DT == STARK_QMM_F32) ((uint32_t*)r.p)[at + i] = w[i % kWords];
            else ((uint16_t*)r.p)[at + i] = (uint16_t)(w[i / 2] >> (16 * (i % 2)));
        }
    }
    QMM_DEVICE float get(int e) const {
        if (DT == STARK_QMM_F32) return __uint_as_float(w[e]);
        const uint32_t h = e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu;
        return DT == STARK_QMM_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
    }
    QMM_DEVICE void set(int e, float a, float b) {  // values e and e + 1, e even
        if (DT == STARK_QMM_F32) w[e] = __float_as_uint(a), w[e + 1] = __float_as_uint(b);
        else if (DT == STARK_QMM_BF16) w[e / 2] = __builtin_bit_cast(uint32_t, bf16x2_t{(__bf16)a, (__bf16)b});
        else w[e / 2] = f32_to_f16_bits(a) | (uint32_t)f32_to_f16_bits(b) << 16;
    }
};

// f64 to f16 through f32, two roundings, as the conversion of a 64-bit tensor does it. The barrier keeps the compiler
// from making one rounding of them.
QMM_DEVICE uint32_t f64_to_f16_bits(double v) {
    float f = (float)v;
    asm("" : "+v"(f));
    return f32_to_f16_bits(f);
}

// v / 15 as a division rounds it: a product with the nearest 1 / 15, off by a step at most, and one correction.
QMM_DEVICE double fifteenth(double v) {
    const double q = v * (1.0 / 15.0);
    return fma(fma(-15.0, q, v), 1.0 / 15.0, q);
}

// The value of another lane of the 16 that share a register row: the lane that CTRL names (quad permutation, or the mirror
// image of 8 or 16 lanes).
template <int CTRL>
QMM_DEVICE uint32_t of_lane(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
QMM_DEVICE float of_lane(float v) {
    return __uint_as_float(of_lane<CTRL>(__float_as_uint(v)));
}
template <int CTRL>
QMM_DEVICE double of_lane(double v) {
    const uint2 w = __builtin_bit_cast(uint2, v);
    return __builtin_bit_cast(double, uint2{of_lane<CTRL>(w.x), of_lane<CTRL>(w.y)});
}
QMM_DEVICE float least(float a, float b) { return fminf(a, b); }
QMM_DEVICE double least(double a, double b) { return fmin(a, b); }
QMM_DEVICE float most(float a, float b) { return fmaxf(a, b); }
QMM_DEVICE double most(double a, double b) { return fmax(a, b); }
template <int CTRL, typename T>
QMM_DEVICE void widen_range(T& lo, T& hi) {
    const T l = of_lane<CTRL>(lo), h = of_lane<CTRL>(hi);
    lo = least(lo, l), hi = most(hi, h);
}

// A row (a head of a token) to DIM / 8 lanes of a wave, eight neighbouring values a lane; a thread does every sets-th
// query head of its token, then key heads, then value heads, with one read of the rotation.
// Keys in f64: a rotated value a c - b s of f32 factors has exact products and one rounding there, and codes, scales and
// biases come out as from exact arithmetic (an f32 sum or quotient beside a half way point would take the wrong code, one
// step of the group's range / 15). Queries of 16 bits in f32, of f32 in f64 as well.
// Bound by latency and vector work together: 2048 tokens of 32 + 2 * 8 heads of 128 (44 MB, 9 us as a copy) take 14.5 us,
// about 170 vector instructions a wave and row (7 us) after two dependent reads (positions, rotation). One row a thread
// took 23 us and all rows as 2^17 or 2^19 threads 16 and 16.5.
template <int DIM, uint32_t DT>
__global__ __launch_bounds__(256) void kv_append(AppendArgs a) {
    constexpr uint32_t L = DIM / 8;  // lanes of a row
    const uint32_t heads = a.heads + 2 * a.cache.kv_heads;
    const uint32_t item = blockIdx.x * (256 / L) + threadIdx.x / L;  // below 2^24 * 32
    const uint32_t l = threadIdx.x % L, d = 8 * l;
    if (item >= a.tokens * a.sets) return;  // whole rows: the lanes of a row leave together
    const uint32_t token = item / a.sets, set = item - token * a.sets;
    const uint32_t pairs = a.rot.pairs;
    const bool turns = d < 2 * pairs;
    // the rotation partner's values: the same eight (interleaved), or those half the rotated width away
    const bool high = !a.rot.interleaved && d >= pairs;
    // A row as this lane holds it: its own values, and its rotation partner's where they are elsewhere. The next row is
    // read before this one is worked on, and the first before the rotation.
    struct Row {
        Eight<DT> x, o;
    };
    const bool elsewhere = turns && !a.rot.interleaved;
    const uint32_t od = high ? d - pairs : d + pairs;
    auto fetch = [&](const KvRows& src, uint32_t head, bool partner) {
        Row r;
        r.x.load(src, token, head, d);
        if (partner) r.o.load(src, token, head, od);
        return r;
    };
    const uint32_t kvh = a.cache.kv_heads, slot = (uint32_t)a.slots[token];
    Row r;
    if (set < a.heads) r = fetch(a.q, set, elsewhere);
    else if (set < a.heads + kvh) r = fetch(a.k, set - a.heads, elsewhere);
    else r.x.load(a.v, token, set - a.heads - kvh, d);
    float2 cs[8];
    if (turns && set < a.heads + a.cache.kv_heads) {
        const uint32_t p0 = a.rot.interleaved ? d / 2 : high ? d - pairs : d;  // this lane's first pair
        const uint32_t np = a.rot.interleaved ? 4 : 8;
        const uint32_t axes = a.rot.axes > 1 ? a.rot.axis8[p0 / 8] >> (2 * (p0 % 8)) : 0;
        const auto position = [&](uint32_t axis) { return (uint32_t)a.rot.positions[axis * a.rot.position_stride + token]; };
        const float2 nan = {__builtin_nanf(""), __builtin_nanf("")};
        if (a.rot.one_axis) {
            const uint32_t pos = position(axes & 3);
            const float4* row = (const float4*)(a.rot.table + (size_t)(pos < a.rot.rows ? pos : 0) * pairs + p0);
            float4 v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = row[(uint32_t)e < np / 2 ? e : 0];
#pragma unroll
            for (int e = 0; e < 4; ++e) cs[2 * e] = float2{v[e].x, v[e].y}, cs[2 * e + 1] = float2{v[e].z, v[e].w};
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (pos >= a.rot.rows) cs[e] = nan;
        } else {
            uint32_t pos[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) pos[e] = position(axes >> (2 * ((uint32_t)e < np ? e : 0)) & 3);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                cs[e] = a.rot.table[(size_t)(pos[e] < a.rot.rows ? pos[e] : 0) * pairs + p0 + ((uint32_t)e < np ? e : 0)];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (pos[e] >= a.rot.rows) cs[e] = nan;
        }
    }
    const uint32_t page = slot >> a.cache.page_shift, page_size = 1u << a.cache.page_shift;
    const bool stored = page < a.cache.page_count;
    const uint32_t in_page = slot & (page_size - 1), t = in_page % kv::kTile;
    uint8_t* const in_cache = a.cache.data + (uint64_t)(stored ? page : 0) * a.cache.page_bytes + in_page / kv::kTile * a.cache.record;
    const uint32_t half_rec = kv::codes_bytes(DIM) + kv::planes_bytes(a.cache.groups), gl = L / a.cache.groups;

    // Scale and bias of the lane's group into a record half, and the lane's eight codes.
    auto quantise = [&](const auto* y, uint8_t* rec) {
        using T = std::remove_cv_t<std::remove_reference_t<decltype(*y)>>;
        // group minimum and maximum; a value that the format does not hold makes the minimum -inf
        T lo = y[0], hi = y[0];
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            lo = least(lo, y[e]), hi = most(hi, y[e]);
            bad |= !(fabs(y[e]) <= (T)kv::kLimit);
        }
        if (bad) lo = -(T)__builtin_inf();
        widen_range<0xb1>(lo, hi);  // lanes 1 0 3 2, then 2 3 0 1: groups of 4 lanes
        widen_range<0x4e>(lo, hi);
        if (gl > 4) widen_range<0x141>(lo, hi);  // mirror of 8 lanes
        if (gl > 8) widen_range<0x140>(lo, hi);  // mirror of 16
        bad = !(lo >= -(T)kv::kLimit);
        const uint32_t sb = bad ? 0x7e00u : f64_to_f16_bits(fifteenth((double)hi - (double)lo));
        const uint32_t bb = bad ? 0x7e00u : f64_to_f16_bits((double)lo);
        const float s = f16_bits_to_f32(sb), b = f16_bits_to_f32(bb);
        if (stored && l % gl == 0) *(uint32_t*)(rec + kv::codes_bytes(DIM) + kv::plane_word(t, l / gl)) = sb | bb << 16;
        uint32_t w = 0;
        if (s > 0.0f) {
            // The code is the nearest step, ties to even, of exact arithmetic. In f32 the quotient is off by less than
            // 2^-18 of its 0 .. 16; where that could matter (within 2^-16 of half way between two codes) f64 decides.
            const float inverse = __builtin_amdgcn_rcpf(s);
            float far = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float t = (float)(y[e] - (T)b) * inverse, n = rintf(t);
                far = fmaxf(far, fabsf(t - n));
                w |= (uint32_t)fminf(fmaxf(n, 0.0f), 15.0f) << (4 * e);
            }
            if (far > 0.5f - 0x1p-16f) {
                w = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) w |= (uint32_t)fmin(fmax(rint(((double)y[e] - (double)b) / (double)s), 0.0), 15.0) << (4 * e);
            }
        }
        return w;
    };
    uint32_t h = set;
    for (; h < a.heads; h += a.sets) {
        const Row now = r;
        if (h + a.sets < a.heads) r = fetch(a.q, h + a.sets, elsewhere);
        Eight<DT> y = now.x;
        if (turns) {
            // 16-bit rows in f32 (they are rounded once more in any case), f32 rows in f64: one rounding, also where the two
            // products nearly cancel
            using T = std::conditional_t<DT == STARK_QMM_F32, double, float>;
            T t[8];
            if (a.rot.interleaved) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const T u = now.x.get(2 * e), v = now.x.get(2 * e + 1), c = cs[e].x, s = cs[e].y;
                    t[2 * e] = fma(u, c, -(v * s)), t[2 * e + 1] = fma(v, c, u * s);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] = fma((T)now.x.get(e), (T)cs[e].x, (T)now.o.get(e) * (T)(high ? cs[e].y : -cs[e].y));
            }
#pragma unroll
            for (int e = 0; e < 8; e += 2) y.set(e, (float)t[e], (float)t[e + 1]);
        }
        y.store(a.q_out, token, h, d);
    }
    h -= a.heads;
    if (set < a.heads && h < kvh) r = fetch(a.k, h, elsewhere);
    for (; h < kvh; h += a.sets) {
        const Row now = r;
        if (h + a.sets < kvh) r = fetch(a.k, h + a.sets, elsewhere);
        // (converted row by row: kept in f64 over the loop they cost a wave of four a SIMD)
#pragma unroll
        for (int e = 0; e < 8; ++e) asm("" : "+v"(cs[e].x), "+v"(cs[e].y));
        double y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = (double)now.x.get(e);
        if (turns) {
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
                    y[e] = fma(y[e], c, (double)now.o.get(e) * s);
                }
            }
        }
        uint8_t* rec = in_cache + (uint64_t)h * a.cache.head_bytes;
        const uint32_t w = quantise(y, rec);
        if (stored) *(uint32_t*)(rec + kv::key_word(DIM, t, l)) = w;
    }
    h -= kvh;
    if (set < a.heads + kvh && h < kvh) r.x.load(a.v, token, h, d);
    for (; h < kvh; h += a.sets) {
        const Eight<DT> now = r.x;
        if (h + a.sets < kvh) r.x.load(a.v, token, h + a.sets, d);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = now.get(e);
        uint8_t* rec = in_cache + (uint64_t)h * a.cache.head_bytes + half_rec;
        const uint32_t w = quantise(y, rec);
        // value bytes: byte i of lane r is byte r % 4 of code word 4 i + r / 4 (of its half of the head). The exchange is
        // of all lanes of the row, whatever it holds.
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
}

// ---------------------------------------------------------------- read

struct ReadArgs {
    KvCache cache;
    KvRows k, v;
    const int32_t* slots;
    uint32_t tokens, sets;
};

// Eight neighbouring values of a head's key and value to a lane, and every sets-th head of a token to a thread. s * code
// + b: the product of an f16 scale and a code is exact in f32, so each value is rounded once (twice to 16 bits). Bound by
// HBM writes: 8192 tokens of 8 heads of 128 to bf16 (43 MB) take 8.8 us, 4.87 TB/s, with two heads a thread; 11.9 with one,
// 11.1 with four, 13.7 with a key's or a value's row a thread.
template <int DIM, uint32_t DT>
__global__ __launch_bounds__(256) void kv_read(ReadArgs a) {
    constexpr uint32_t L = DIM / 8;
    const uint32_t item = blockIdx.x * (256 / L) + threadIdx.x / L, l = threadIdx.x % L;
    if (item >= a.tokens * a.sets) return;
    const uint32_t token = item / a.sets, set = item - token * a.sets;
    const uint32_t slot = (uint32_t)a.slots[token];
    const uint32_t page = slot >> a.cache.page_shift, page_size = 1u << a.cache.page_shift;
    if (page >= a.cache.page_count) return;
    const uint32_t in_page = slot & (page_size - 1), t = in_page % kv::kTile;
    const uint8_t* const in_cache = a.cache.data + (uint64_t)page * a.cache.page_bytes + in_page / kv::kTile * a.cache.record;
    const uint32_t half_rec = kv::codes_bytes(DIM) + kv::planes_bytes(a.cache.groups);
    const uint32_t plane_at = kv::codes_bytes(DIM) + kv::plane_word(t, l * a.cache.groups / L);
    const uint32_t key_at = kv::key_word(DIM, t, l);
    const uint32_t value_at = DIM == 64 ? kv::value_byte(DIM, t, 0, 2 * l, 0) : kv::value_byte(DIM, t, l / 16, l % 16, 0);
    const int row = (int)(threadIdx.x & 63) - (int)l;
    auto write = [&](const KvRows& dst, uint32_t head, uint32_t w, uint32_t plane) {
        const float s = f16_bits_to_f32(plane & 0xffffu), b = f16_bits_to_f32(plane >> 16);
        Eight<DT> out;
#pragma unroll
        for (int e = 0; e < 8; e += 2)
            out.set(e, fmaf(s, (float)(w >> (4 * e) & 15u), b), fmaf(s, (float)(w >> (4 * e + 4) & 15u), b));
        if (dst.p) out.store(dst, token, head, 8 * l);
    };
    for (uint32_t head = set; head < a.cache.kv_heads; head += a.sets) {
        const uint8_t* rec = in_cache + (uint64_t)head * a.cache.head_bytes;
        const uint32_t k = *(const uint32_t*)(rec + key_at), kp = *(const uint32_t*)(rec + plane_at);
        uint32_t u;
        if (DIM == 64)  // rows of 8 bytes for four tokens
            u = *(const uint16_t*)(rec + half_rec + value_at) | (uint32_t)*(const uint16_t*)(rec + half_rec + value_at + 8) << 16;
        else
            u = *(const uint32_t*)(rec + half_rec + value_at);
        const uint32_t vp = *(const uint32_t*)(rec + half_rec + plane_at);
        write(a.k, head, k, kp);
        // the value's bytes are spread as kv_append puts them: code byte m of lane l is byte i of word 4 (l % 4) + m
        uint32_t v = 0;
#pragma unroll
        for (uint32_t m = 0; m < 4; ++m) {
            const uint32_t from = DIM == 64 ? 2 * (l % 4) + m / 2 : l / 16 * 16 + 4 * (l % 4) + m;
            const uint32_t byte = DIM == 64 ? 2 * (m % 2) + l / 4 : l % 16 / 4;
            v |= ((uint32_t)__shfl((int)u, row + (int)from, 64) >> (8 * byte) & 0xffu) << (8 * m);
        }
        write(a.v, head, v, vp);
    }
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

template <uint32_t DT>
void append_launch(dim3 grid, hipStream_t s, const AppendArgs& a) {
    if (a.cache.dim == 64) hipLaunchKernelGGL((kv_append<64, DT>), grid, dim3(256), 0, s, a);
    else if (a.cache.dim == 128) hipLaunchKernelGGL((kv_append<128, DT>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((kv_append<256, DT>), grid, dim3(256), 0, s, a);
}

template <uint32_t DT>
void read_launch(dim3 grid, hipStream_t s, const ReadArgs& a) {
    if (a.cache.dim == 64) hipLaunchKernelGGL((kv_read<64, DT>), grid, dim3(256), 0, s, a);
    else if (a.cache.dim == 128) hipLaunchKernelGGL((kv_read<128, DT>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((kv_read<256, DT>), grid, dim3(256), 0, s, a);
}

uint32_t sets_of(uint32_t tokens, uint32_t heads, uint32_t dim) {
    const uint32_t each = kv::rows_each((uint64_t)tokens * heads * (dim / 8));
    return (heads + each - 1) / each;
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
    // what is written overlaps nothing else: workgroups read while others write
    const uint64_t words[] = {p->batch, p->batch, p->free_capacity, 1, (uint64_t)p->batch * p->table_stride, p->batch + 1ull,
                              p->batch, p->token_capacity, p->token_capacity, 1, 1};
    for (int i = 4; i < 11; ++i)
        for (int j = 0; j < 11; ++j) {
            const uintptr_t x = (uintptr_t)all[i], y = (uintptr_t)all[j];
            if (i != j && words[i] && words[j] && x < y + 4 * words[j] && y < x + 4 * words[i]) return STARK_QMM_INVALID_ARGUMENT;
        }
    PlanArgs a{p->cached, p->added, p->free_pages, p->free_count, p->block_table, p->query_start, p->kv_lengths, p->slots,
               p->positions, p->free_left, p->status, p->batch, p->token_capacity, p->free_capacity, p->table_stride, 4};
    while ((1u << a.page_shift) < p->page_size) ++a.page_shift;
    const uint32_t blocks = std::max(1u, (p->token_capacity + kPlanThreads - 1) / kPlanThreads);
    if (p->batch <= kPlanThreads) hipLaunchKernelGGL(kv_plan<1>, dim3(blocks), dim3(kPlanThreads), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(kv_plan<4>, dim3(blocks), dim3(kPlanThreads), 0, (hipStream_t)stream, a);
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
    if (p->q && p->q == p->q_out && ((p->tokens > 1 && p->q_token_stride != p->q_out_token_stride) ||
                                     (heads > 1 && p->q_head_stride != p->q_out_head_stride)))
        return STARK_QMM_INVALID_ARGUMENT;  // a row would be written where another is still to be read
    const stark_qmm_rotary& r = p->rotary;
    if (r.rotary_dim) {
        if (r.rotary_dim % 16 || r.rotary_dim > dim || r.axes < 1 || r.axes > 4) return STARK_QMM_INVALID_ARGUMENT;
        if (!r.table || !kv_aligned(r.table, 8) || !r.positions || !kv_aligned(r.positions, 4) ||
            r.table_rows == 0 || r.table_rows > 0x7fffffffu || (r.axes > 1 && (r.position_stride < p->tokens || r.position_stride >> 32)))
            return STARK_QMM_INVALID_ARGUMENT;
        a.rot = Rotary{(const float2*)r.table, r.positions, r.axes > 1 ? r.position_stride : 0, r.table_rows,
                       r.rotary_dim / 2, r.axes, r.interleaved != 0, kv_aligned(r.table, 16), {}};
        for (uint32_t i = 0; i < a.rot.pairs; ++i) {
            if (r.axis_of_pair[i] >= r.axes) return STARK_QMM_INVALID_ARGUMENT;
            a.rot.axis8[i / 8] |= (uint16_t)(r.axis_of_pair[i] << (2 * (i % 8)));
            if (r.axis_of_pair[i] != r.axis_of_pair[i / 8 * 8]) a.rot.one_axis = 0;
        }
    }
    a.q = kv_rows(p->q, p->q_token_stride, p->q_head_stride, dt);
    a.q_out = kv_rows(p->q_out, p->q_out_token_stride, p->q_out_head_stride, dt);
    a.k = kv_rows(p->k, p->k_token_stride, p->k_head_stride, dt);
    a.v = kv_rows(p->v, p->v_token_stride, p->v_head_stride, dt);
    a.slots = p->slots;
    a.tokens = p->tokens, a.heads = heads;
    a.sets = sets_of(p->tokens, heads + 2 * a.cache.kv_heads, dim);
    const hipStream_t s = (hipStream_t)stream;
    return launch_rows(dim, (uint64_t)p->tokens * a.sets, [&](dim3 grid) {
        if (dt == STARK_QMM_F32) append_launch<STARK_QMM_F32>(grid, s, a);
        else if (dt == STARK_QMM_F16) append_launch<STARK_QMM_F16>(grid, s, a);
        else append_launch<STARK_QMM_BF16>(grid, s, a);
    });
}

stark_qmm_status stark_qmm_kv_read(const stark_qmm_kv_read_args* p, void* stream) {
    if (!p) return STARK_QMM_INVALID_ARGUMENT;
    if (p->struct_size != sizeof(*p)) return STARK_QMM_ABI_MISMATCH;
    ReadArgs a{};
    const stark_qmm_status st = kv_view(p->cache, &a.cache);
    if (st != STARK_QMM_OK) return st;
    if (!dt_ok(p->data_type)) return STARK_QMM_UNSUPPORTED_DATA_TYPE;
    if (p->tokens > (1u << 24)) return STARK_QMM_INVALID_ARGUMENT;
    if (p->tokens == 0) return STARK_QMM_OK;
    if ((!p->k && !p->v) || !p->slots || !kv_aligned(p->slots, 4)) return STARK_QMM_INVALID_ARGUMENT;
    const uint32_t dim = a.cache.dim, dt = p->data_type;
    if ((p->k && !kv_rows_ok(p->k, p->k_token_stride, p->k_head_stride, p->tokens, a.cache.kv_heads, dim, dt)) ||
        (p->v && !kv_rows_ok(p->v, p->v_token_stride, p->v_head_stride, p->tokens, a.cache.kv_heads, dim, dt)))
        return STARK_QMM_INVALID_ARGUMENT;
    a.k = kv_rows(p->k, p->k_token_stride, p->k_head_stride, dt);
    a.v = kv_rows(p->v, p->v_token_stride, p->v_head_stride, dt);
    a.slots = p->slots;
    a.tokens = p->tokens;
    const hipStream_t s = (hipStream_t)stream;
    a.sets = (a.cache.kv_heads + 1) / 2;
    return launch_rows(dim, (uint64_t)p->tokens * a.sets, [&](dim3 grid) {
        if (dt == STARK_QMM_F32) read_launch<STARK_QMM_F32>(grid, s, a);
        else if (dt == STARK_QMM_F16) read_launch<STARK_QMM_F16>(grid, s, a);
        else read_launch<STARK_QMM_BF16>(grid, s, a);
    });
}

}  // extern "C"
