// Checks shared by the entry points of the 4-bit paged key/value cache.
#pragma once

#include "qmm_common.h"

#include "kv_layout.h"

namespace qmm {

// The cache as the kernels see it.
struct KvCache {
    uint8_t* data;
    uint32_t page_count, page_shift, kv_heads, dim, groups, record;
    uint32_t head_bytes, page_bytes;  // of one head's records in a page, and of a page
};

inline bool kv_aligned(const void* p, uint64_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// Geometry checks; fills `out` but for data.
inline stark_qmm_status kv_geometry(const stark_qmm_kv_cache& c, KvCache* out, uint64_t* bytes) {
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return STARK_QMM_UNSUPPORTED;
    if ((c.group_size != 32 && c.group_size != 64 && c.group_size != 128) || c.head_dim % c.group_size)
        return STARK_QMM_UNSUPPORTED_GROUP_SIZE;
    if (c.page_size < 16 || c.page_size > 1024 || (c.page_size & (c.page_size - 1))) return STARK_QMM_INVALID_ARGUMENT;
    if (c.page_count == 0 || c.kv_heads == 0 || c.kv_heads > 1024) return STARK_QMM_INVALID_ARGUMENT;
    if ((uint64_t)c.page_count * c.page_size > 0x7fffffffull) return STARK_QMM_INVALID_ARGUMENT;
    const uint32_t groups = c.head_dim / c.group_size;
    uint32_t shift = 4;
    while ((1u << shift) < c.page_size) ++shift;
    const uint32_t record = kv::record_bytes(c.head_dim, groups), head = c.page_size / kv::kTile * record;
    // a page is at most 1024 heads * 64 records * 5120 bytes, below 2^32
    *out = KvCache{nullptr, c.page_count, shift, c.kv_heads, c.head_dim, groups, record, head, c.kv_heads * head};
    *bytes = (uint64_t)c.page_count * out->page_bytes;
    return STARK_QMM_OK;
}

inline stark_qmm_status kv_view(const stark_qmm_kv_cache& c, KvCache* out) {
    uint64_t bytes;
    const stark_qmm_status st = kv_geometry(c, out, &bytes);
    if (st != STARK_QMM_OK) return st;
    if (!c.data || !kv_aligned(c.data, 128)) return STARK_QMM_INVALID_ARGUMENT;
    if (c.data_size < bytes) return STARK_QMM_UNSUPPORTED_LAYOUT;
    out->data = (uint8_t*)c.data;
    return STARK_QMM_OK;
}

inline uint64_t kv_element(uint32_t dt) { return dt == STARK_QMM_F32 ? 4 : 2; }

// Rows [tokens, heads, dim] with strides in elements, as kernels see them.
struct KvRows {
    const void* p;
    uint64_t token, head;
    uint32_t vec;  // every row starts 16-byte aligned
};

inline KvRows kv_rows(const void* p, uint64_t token, uint64_t head, uint32_t dt) {
    const uint64_t e = kv_element(dt);
    return {p, token, head, (uint32_t)(kv_aligned(p, 16) && token * e % 16 == 0 && head * e % 16 == 0)};
}

// The pointer is aligned to its type, heads do not overlap, nor do tokens (a single token or head has no stride).
inline bool kv_rows_ok(const void* p, uint64_t token, uint64_t head, uint32_t tokens, uint32_t heads, uint32_t dim,
                       uint32_t dt) {
    if (!p || !kv_aligned(p, kv_element(dt))) return false;
    if (token >> 40 || head >> 40) return false;
    const uint64_t ht = heads > 1 ? head : dim, span = (uint64_t)(heads - 1) * ht + dim;
    if (ht < dim) return false;
    if (tokens <= 1) return true;
    // tokens outside heads ([tokens, heads, dim]), or heads outside tokens ([heads, tokens, dim])
    return token >= span || (token >= dim && heads > 1 && head >= (uint64_t)(tokens - 1) * token + dim);
}

}  // namespace qmm
