// Entry points of attention over the 4-bit paged key/value cache: checks, and which kernel takes which requests.
#include <atomic>

#include "kv_attend.h"

namespace {

using namespace qmm;

// Checks all but the pointers, which a size query need not have; fills the lengths.
stark_qmm_status check(const stark_qmm_kv_attention_args* p, AttendArgs* a) {
    if (!p) return STARK_QMM_INVALID_ARGUMENT;
    if (p->struct_size != sizeof(*p)) return STARK_QMM_ABI_MISMATCH;
    uint64_t bytes;
    const stark_qmm_status st = kv_geometry(p->cache, &a->cache, &bytes);
    if (st != STARK_QMM_OK) return st;
    if (p->data_type != STARK_QMM_F16 && p->data_type != STARK_QMM_BF16) return STARK_QMM_UNSUPPORTED_DATA_TYPE;
    if (p->heads == 0 || p->heads > 65536 || p->heads % a->cache.kv_heads) return STARK_QMM_INVALID_ARGUMENT;
    if (p->batch > (1u << 20) || p->tokens > (1u << 24) || p->max_kv > 0x7fffffffu) return STARK_QMM_INVALID_ARGUMENT;
    if ((uint64_t)p->table_stride * p->cache.page_size > 0x7fffffffull || p->table_stride == 0)
        return STARK_QMM_INVALID_ARGUMENT;
    if (!(p->soft_cap == 0.0f || (p->soft_cap >= 0x1p-20f && p->soft_cap <= 0x1p20f)) ||
        !(p->scale == 0.0f || (fabsf(p->scale) >= 0x1p-64f && fabsf(p->scale) <= 0x1p64f)))
        return STARK_QMM_INVALID_ARGUMENT;
    a->batch = p->batch, a->tokens = p->tokens, a->heads = p->heads, a->ratio = p->heads / a->cache.kv_heads;
    a->stride = p->table_stride;
    a->max_query = std::min(p->max_query, p->tokens);
    a->max_kv = std::min(p->max_kv, p->table_stride * p->cache.page_size);
    if (a->max_kv > 0x7fff0000u) return STARK_QMM_INVALID_ARGUMENT;  // positions past a tile's end are int32 as well
    a->is_bf16 = p->data_type == STARK_QMM_BF16;
    a->causal = p->causal != 0, a->window = (int32_t)std::min(p->window, 0x7fffffffu);
    const float scale = p->scale == 0.0f ? 1.0f : fabsf(p->scale);
    a->sign = p->scale == 0.0f ? 0.0f : p->scale < 0.0f ? -1.0f : 1.0f;
    a->scale = p->soft_cap != 0.0f ? 2.0f * kLog2e * scale / p->soft_cap : kLog2e * scale;
    a->cap = p->soft_cap * kLog2e;
    return STARK_QMM_OK;
}

// Compute units of the current device, asked for once.
stark_qmm_status compute_units(uint32_t* cus) {
    static std::atomic<int> known[64];
    int dev = 0;
    QMM_HIP_CHECK(hipGetDevice(&dev));
    int n = dev < 64 ? known[dev].load(std::memory_order_relaxed) : 0;
    if (n == 0) {
        QMM_HIP_CHECK(hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev));
        if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
    }
    *cus = (uint32_t)n;
    return STARK_QMM_OK;
}

// How the checked call's work is dealt, and the bytes that its partial results need.
stark_qmm_status plan_work(AttendArgs* a, uint64_t* workspace) {
    *workspace = 0;
    if (a->batch == 0 || a->max_query == 0) return STARK_QMM_OK;  // (tiling divides by the requests)
    const kv::Rows rows = kv::row_limit(a->batch, a->max_query, a->ratio, a->max_kv);
    const uint64_t most = (uint64_t)a->max_query * a->ratio, all = (uint64_t)a->tokens * a->ratio;
    a->row_limit = std::min<uint64_t>(rows.limit, most), a->row_block = rows.block;
    const uint32_t blocks = (a->row_limit + a->row_block - 1) / a->row_block;
    // all refusals are here: none after a launch
    if (!kv::fits(a->batch, a->cache.kv_heads, blocks, a->max_kv, most > a->row_limit ? all : 0)) return STARK_QMM_UNSUPPORTED;
    uint32_t cus = 0;
    const stark_qmm_status st = compute_units(&cus);
    if (st != STARK_QMM_OK) return st;
    if (a->row_limit) {
        a->ratio_inverse = (65535 + a->ratio) / a->ratio;
        const kv::Share w = kv::share(a->batch, a->cache.kv_heads * blocks, a->row_block, a->max_kv,
                                      cus * (a->cache.dim == 256 ? 1 : 2));
        a->whole = w.whole, a->grid = w.grid;
        a->inverse = w.grid > 1 ? (uint32_t)((1ull << 32) / w.grid) : 0xffffffffu;
        if (!w.whole) *workspace = (uint64_t)w.grid * (2 * kRows * (a->cache.dim * 4ull + 8) + 16);
    }
    if (most > a->row_limit) {
        const kv::Tiling t = kv::tiling(a->batch, a->cache.kv_heads, all, most, a->max_kv, cus);
        const uint64_t even = (uint64_t)t.tiles * a->batch, need = kv::row_tiles(all, a->batch);
        a->tiles = even <= need ? t.tiles : 0, a->turns = (uint32_t)std::min(even, need);
        a->pieces = t.pieces;
        if (t.pieces > 1) *workspace += (uint64_t)a->tokens * a->heads * t.pieces * (a->cache.dim * 4ull + 8);
    }
    return STARK_QMM_OK;
}

}  // namespace

extern "C" {

stark_qmm_status stark_qmm_kv_attention_workspace_size(const stark_qmm_kv_attention_args* args, uint64_t* bytes) {
    AttendArgs a{};
    if (!bytes) return STARK_QMM_INVALID_ARGUMENT;
    const stark_qmm_status st = check(args, &a);
    return st != STARK_QMM_OK ? st : plan_work(&a, bytes);
}

stark_qmm_status stark_qmm_kv_attention(const stark_qmm_kv_attention_args* p, void* stream) {
    AttendArgs a{};
    stark_qmm_status st = check(p, &a);
    if (st != STARK_QMM_OK) return st;
    st = kv_view(p->cache, &a.cache);
    if (st != STARK_QMM_OK) return st;
    if (a.batch == 0 || a.max_query == 0) return STARK_QMM_OK;
    if (!p->query_start || !p->kv_lengths || !p->block_table || !kv_aligned(p->query_start, 4) ||
        !kv_aligned(p->kv_lengths, 4) || !kv_aligned(p->block_table, 4) || !kv_aligned(p->lse, 4))
        return STARK_QMM_INVALID_ARGUMENT;
    if (!kv_rows_ok(p->q, p->q_token_stride, p->q_head_stride, a.tokens, a.heads, a.cache.dim, p->data_type) ||
        !kv_rows_ok(p->out, p->out_token_stride, p->out_head_stride, a.tokens, a.heads, a.cache.dim, p->data_type))
        return STARK_QMM_INVALID_ARGUMENT;
    if (p->q == p->out) return STARK_QMM_INVALID_ARGUMENT;  // workgroups read rows that others would have written
    uint64_t need = 0;
    st = plan_work(&a, &need);
    if (st != STARK_QMM_OK) return st;
    if (need && (!p->workspace || !kv_aligned(p->workspace, 16))) return STARK_QMM_INVALID_ARGUMENT;
    if (need > p->workspace_size) return STARK_QMM_WORKSPACE_TOO_SMALL;
    a.q = kv_rows(p->q, p->q_token_stride, p->q_head_stride, p->data_type);
    a.out = kv_rows(p->out, p->out_token_stride, p->out_head_stride, p->data_type);
    a.lse = p->lse;
    a.table = p->block_table, a.query_start = p->query_start, a.kv_lengths = p->kv_lengths;
    if (need) {
        uint8_t* p0 = (uint8_t*)p->workspace;
        if (a.row_limit && !a.whole) {
            a.begun = (int4*)p0;
            a.po = (float*)(a.begun + a.grid);
            a.pml = (float2*)(a.po + 2ull * a.grid * kRows * a.cache.dim);
            p0 = (uint8_t*)(a.pml + 2ull * a.grid * kRows);
        }
        a.tile_po = (float*)p0;
        a.tile_pml = (float2*)(a.tile_po + (uint64_t)a.tokens * a.heads * a.pieces * a.cache.dim);
    }
    const hipStream_t s = (hipStream_t)stream;
    if (a.row_limit) {
        st = launch_attend_rows(a, s);
        if (st != STARK_QMM_OK) return st;
    }
    return (uint64_t)a.max_query * a.ratio > a.row_limit ? launch_attend_tiles(a, s) : STARK_QMM_OK;
}

}  // extern "C"
