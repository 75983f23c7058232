// Entry points of the products of 8-bit floating-point codes: checks, and which kernel takes a call.
#include "fp8_common.h"

namespace {

using namespace qmm;

constexpr uint64_t kStride = 1ull << 24, kScaleStride = 1ull << 22, kFar = 1ull << 40;

struct Groups {  // of a dense call: one
    uint32_t experts = 1;
    uint64_t b_expert = 0, bs_expert = 0, bias_expert = 0;
    bool gathered = false;
    uint32_t a_row_count = 0;
};

// A row stride in bytes; of a single row it has no meaning.
bool code_rows(uint64_t rows, uint64_t stride, uint32_t k) { return rows <= 1 || (stride % 16 == 0 && stride >= k && stride <= kStride); }

// All but the pointers, which a size query need not have.
stark_qmm_status check_sizes(const stark_qmm_fp8_matmul_args& q, const Groups& g, Fp8Product* p) {
    if (q.struct_size != sizeof(q)) return STARK_QMM_ABI_MISMATCH;
    if (!fp8_type(q.d_type)) return STARK_QMM_UNSUPPORTED_DATA_TYPE;
    if (q.d_ops.rht_factors) return STARK_QMM_UNSUPPORTED_D_OP;
    if (q.m > (1u << 24) || q.n > (1u << 24) || q.k == 0 || q.k > (1u << 20)) return STARK_QMM_INVALID_ARGUMENT;
    if (g.experts == 0 || g.experts > 1024) return STARK_QMM_INVALID_ARGUMENT;
    const uint64_t a_rows = g.gathered ? g.a_row_count : q.m;
    if (g.gathered && (g.a_row_count == 0 || g.a_row_count > 0x7fffffffu)) return STARK_QMM_INVALID_ARGUMENT;
    if (!code_rows(a_rows, q.a_row_stride, q.k) || !code_rows(q.n, q.b_row_stride, q.k)) return STARK_QMM_INVALID_ARGUMENT;
    if (q.a_scale_row_stride > kScaleStride || q.a_scale_block_stride >> 32 || q.b_scale_row_stride >> 32 || q.b_scale_block_stride >> 32 ||
        q.d_row_stride > kFar)
        return STARK_QMM_INVALID_ARGUMENT;
    if (q.m > 1 && q.d_row_stride < q.n) return STARK_QMM_INVALID_ARGUMENT;
    if (g.experts > 1) {
        if (g.b_expert % 16 || g.b_expert > kFar || g.bs_expert > kFar || g.bias_expert > kFar) return STARK_QMM_INVALID_ARGUMENT;
    }
    p->a_stride = a_rows <= 1 ? 0 : q.a_row_stride, p->b_stride = q.n <= 1 ? 0 : q.b_row_stride;
    p->as_row = a_rows <= 1 ? 0 : q.a_scale_row_stride, p->as_block = q.a_scale_block_stride;
    p->bs_row = q.b_scale_row_stride, p->bs_block = q.b_scale_block_stride;
    p->b_expert = g.b_expert, p->bs_expert = g.bs_expert, p->bias_expert = g.bias_expert;
    p->d_stride = q.m <= 1 ? q.n : q.d_row_stride;
    p->m = q.m, p->n = q.n, p->k = q.k, p->experts = g.experts, p->a_row_count = g.gathered ? g.a_row_count : q.m;
    p->d_dt = q.d_type, p->ab_scale = q.d_ops.ab_scale, p->soft_cap = q.d_ops.soft_cap;
    p->flags = (q.d_ops.accumulate ? FLAG_ACCUMULATE : 0u) | (q.d_ops.has_soft_cap ? FLAG_SOFT_CAP : 0u);
    // a gathered row's place is a 32-bit offset from the first
    if (g.gathered && (fp8_span(a_rows, p->a_stride, (q.k + 15) / 16 * 16) >> 32 || fp8_span(a_rows, 4 * p->as_row, 4) >> 32))
        return STARK_QMM_UNSUPPORTED;
    return STARK_QMM_OK;
}

// Which kernel takes a call of some outputs.
stark_qmm_status choice(const Fp8Product& p, bool grouped, fp8::Choice* c) {
    *c = fp8::choose(p.m, p.n, p.k, p.experts, grouped, fp8_exact(p.d_dt));
    return fp8::workgroups(*c, p.m, p.n, p.k, p.experts) > fp8::kMostGroups ? STARK_QMM_UNSUPPORTED : STARK_QMM_OK;
}

// The parts' sums: rows of whole 16-byte pieces.
uint64_t partial_stride(const Fp8Product& p) { return (p.n + 3ull) / 4 * 4; }
uint64_t workspace_of(const Fp8Product& p, fp8::Choice c) { return c.parts > 1 ? 4ull * c.parts * p.m * partial_stride(p) : 0; }

stark_qmm_status size_of(const stark_qmm_fp8_matmul_args& q, const Groups& g, bool grouped, uint64_t* bytes) {
    Fp8Product p{};
    fp8::Choice c{0, 16, 1};
    stark_qmm_status st = check_sizes(q, g, &p);
    if (st == STARK_QMM_OK && p.m && p.n) st = choice(p, grouped, &c);
    if (st == STARK_QMM_OK) *bytes = workspace_of(p, c);
    return st;
}

stark_qmm_status run(const stark_qmm_fp8_matmul_args& q, const Groups& g, const int32_t* start, const int32_t* rows, hipStream_t stream) {
    Fp8Product p{};
    stark_qmm_status st = check_sizes(q, g, &p);
    if (st != STARK_QMM_OK) return st;
    if (q.m == 0 || q.n == 0) return STARK_QMM_OK;
    fp8::Choice c;
    st = choice(p, start != nullptr, &c);
    if (st != STARK_QMM_OK) return st;
    const uint64_t e = fp8_element(q.d_type), wide = ((uint64_t)q.k + 15) / 16 * 16, kb = fp8::blocks(q.k), nb = fp8::blocks(q.n);
    if (!q.a || !q.a_scales || !q.b || !q.b_scales || !q.d) return STARK_QMM_INVALID_ARGUMENT;
    if (!fp8_aligned(q.a, 16) || !fp8_aligned(q.b, 16) || !fp8_aligned(q.a_scales, 4) || !fp8_aligned(q.b_scales, 4) ||
        !fp8_aligned(q.d, e) || !fp8_aligned(q.d_ops.bias, e) || !fp8_aligned(start, 4) || !fp8_aligned(rows, 4))
        return STARK_QMM_INVALID_ARGUMENT;
    // what d must not meet
    const uint64_t last = g.experts - 1, dn = e * fp8_span(q.m, p.d_stride, q.n), an = fp8_span(p.a_row_count, p.a_stride, wide),
                   asn = 4 * (fp8_span(p.a_row_count, p.as_row, 1) + (kb - 1) * p.as_block), bn = last * g.b_expert + fp8_span(q.n, p.b_stride, wide),
                   bsn = 4 * (last * g.bs_expert + fp8_span(nb, p.bs_row, 1) + (kb - 1) * p.bs_block);
    if (fp8_overlap(q.d, dn, q.a, an) || fp8_overlap(q.d, dn, q.a_scales, asn) || fp8_overlap(q.d, dn, q.b, bn) ||
        fp8_overlap(q.d, dn, q.b_scales, bsn) || fp8_overlap(q.d, dn, q.d_ops.bias, e * (last * g.bias_expert + q.n)) ||
        fp8_overlap(q.d, dn, start, 4ull * (g.experts + 1)) || fp8_overlap(q.d, dn, rows, 4ull * q.m))
        return STARK_QMM_INVALID_ARGUMENT;
    p.a = q.a, p.b = q.b, p.as = q.a_scales, p.bs = q.b_scales, p.d = q.d, p.bias = q.d_ops.bias;
    p.group_start = start, p.a_rows = rows;
    p.vec = fp8_aligned(q.d, 4 * e) && p.d_stride % 4 == 0;
    p.plain = e == 2 && !p.flags && !p.bias && fp8_aligned(q.d, 16) && p.d_stride % 8 == 0;
    p.parts = c.parts;
    const uint64_t need = workspace_of(p, c);
    if (need) {
        if (!q.workspace || !fp8_aligned(q.workspace, 16)) return STARK_QMM_INVALID_ARGUMENT;
        if (need > q.workspace_size) return STARK_QMM_WORKSPACE_TOO_SMALL;
        if (fp8_overlap(q.workspace, need, q.d, dn) || fp8_overlap(q.workspace, need, q.a, an) || fp8_overlap(q.workspace, need, q.b, bn) ||
            fp8_overlap(q.workspace, need, q.a_scales, asn) || fp8_overlap(q.workspace, need, q.b_scales, bsn) ||
            fp8_overlap(q.workspace, need, q.d_ops.bias, e * q.n))
            return STARK_QMM_INVALID_ARGUMENT;
        p.partial = (float*)q.workspace, p.partial_stride = partial_stride(p);
    }
    return c.tile ? launch_fp8_tiles(p, c.tile, stream) : launch_fp8_rows(p, c.rows, stream);
}

stark_qmm_status groups_of(const stark_qmm_fp8_grouped_args* a, Groups* g) {
    if (!a) return STARK_QMM_INVALID_ARGUMENT;
    if (a->struct_size != sizeof(*a)) return STARK_QMM_ABI_MISMATCH;
    g->experts = a->experts, g->b_expert = a->b_expert_stride, g->bs_expert = a->b_scale_expert_stride;
    g->bias_expert = a->bias_expert_stride, g->gathered = a->a_rows != nullptr, g->a_row_count = a->a_row_count;
    return STARK_QMM_OK;
}

}  // namespace

extern "C" {

stark_qmm_status stark_qmm_fp8_matmul_workspace_size(const stark_qmm_fp8_matmul_args* args, uint64_t* bytes) {
    if (!args || !bytes) return STARK_QMM_INVALID_ARGUMENT;
    return size_of(*args, Groups{}, false, bytes);
}

stark_qmm_status stark_qmm_fp8_matmul(const stark_qmm_fp8_matmul_args* args, void* stream) {
    if (!args) return STARK_QMM_INVALID_ARGUMENT;
    return run(*args, Groups{}, nullptr, nullptr, (hipStream_t)stream);
}

stark_qmm_status stark_qmm_fp8_grouped_matmul_workspace_size(const stark_qmm_fp8_grouped_args* args, uint64_t* bytes) {
    if (!bytes) return STARK_QMM_INVALID_ARGUMENT;
    Groups g;
    const stark_qmm_status st = groups_of(args, &g);
    return st != STARK_QMM_OK ? st : size_of(args->product, g, true, bytes);
}

stark_qmm_status stark_qmm_fp8_grouped_matmul(const stark_qmm_fp8_grouped_args* args, void* stream) {
    Groups g;
    const stark_qmm_status st = groups_of(args, &g);
    if (st != STARK_QMM_OK) return st;
    if (args->product.m && args->product.n && !args->group_start) return STARK_QMM_INVALID_ARGUMENT;
    return run(args->product, g, args->group_start, args->a_rows, (hipStream_t)stream);
}

}  // extern "C"
