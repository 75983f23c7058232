"""Index arithmetic of the 4-bit key/value cache (csrc/kv_layout.h, compiled for the CPU), and what the entry points
refuse before they touch a GPU."""
import ctypes as C
import functools
import os
import random
import subprocess
import tempfile

import numpy as np
import pytest

from tests import kv_ref as R

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stark_amd", "csrc")

_WRAP = """
#include "kv_layout.h"
extern "C" {
uint32_t record_bytes(uint32_t d, uint32_t g) { return kv::record_bytes(d, g); }
uint32_t key_word(uint32_t dim, uint32_t t, uint32_t d) { return kv::key_word(dim, t, d); }
uint32_t value_byte(uint32_t dim, uint32_t t, uint32_t h, uint32_t r, uint32_t i) { return kv::value_byte(dim, t, h, r, i); }
uint32_t plane_word(uint32_t t, uint32_t g) { return kv::plane_word(t, g); }
uint64_t record_index(uint64_t p, uint32_t n, uint32_t h, uint32_t s, uint32_t at) { return kv::record_index(p, n, h, s, at); }
void visible(int32_t i, int32_t q, int32_t k, int c, int32_t w, int32_t* r) {
    const kv::Range x = kv::visible(i, q, k, c != 0, w); r[0] = x.lo; r[1] = x.hi;
}
void request_range(int32_t q, int32_t k, int c, int32_t w, int32_t* r) {
    const kv::Range x = kv::request_range(q, k, c != 0, w); r[0] = x.lo; r[1] = x.hi;
}
void request(int32_t s, int32_t e, int32_t k, uint32_t n, uint32_t mq, uint32_t mk, int32_t* r) {
    const kv::Request x = kv::request(s, e, k, n, mq, mk); r[0] = x.first; r[1] = x.q_len; r[2] = x.kv_len;
}
void page_plan(int64_t c, int64_t a, uint32_t s, uint32_t w, int32_t* r) {
    const kv::PagePlan x = kv::page_plan(c, a, s, w); r[0] = x.before; r[1] = x.need;
}
void share(uint32_t batch, uint32_t heads, uint32_t block, uint32_t max_kv, uint32_t slots, uint32_t* r) {
    const kv::Share x = kv::share(batch, heads, block, max_kv, slots); r[0] = x.whole; r[1] = x.grid;
}
uint32_t share_of(uint32_t total, uint32_t grid, uint32_t keys) {
    return kv::share_of(total, grid, grid > 1 ? (uint32_t)((1ull << 32) / grid) : 0xffffffffu, keys);
}
void row_limit(uint32_t b, uint32_t q, uint32_t r, uint32_t kv, uint32_t* o) { const kv::Rows x = kv::row_limit(b, q, r, kv); o[0] = x.limit; o[1] = x.block; }
int32_t piece_keys(int32_t range, uint32_t pieces) { return kv::piece_keys(range, pieces); }
void tiling(uint32_t batch, uint32_t heads, uint64_t rows, uint64_t most, uint32_t max_kv, uint32_t cus, uint32_t* o) {
    const kv::Tiling t = kv::tiling(batch, heads, rows, most, max_kv, cus); o[0] = t.tiles; o[1] = t.pieces;
}
uint32_t unit_keys(uint32_t block) { return kv::unit_keys(block); }
}
"""


@functools.lru_cache(None)
def rules():
    with tempfile.TemporaryDirectory() as d:
        src, lib = os.path.join(d, "kv.cpp"), os.path.join(d, "kv.so")
        with open(src, "w") as f:
            f.write(_WRAP)
        subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", CSRC, src, "-o", lib], check=True)
        r = C.CDLL(lib)
        r.record_index.restype = C.c_uint64
        r.record_index.argtypes = [C.c_uint64] + [C.c_uint32] * 4
        r.page_plan.argtypes = [C.c_int64, C.c_int64, C.c_uint32, C.c_uint32, C.c_void_p]
        return r


def _out(fn, n, *args, kind=C.c_int32):
    r = (kind * n)()
    fn(*args, r)
    return tuple(r)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_every_code_and_plane_has_a_place_of_its_own(dim):
    L = rules()
    keys = {L.key_word(dim, t, d) for t in range(16) for d in range(dim // 8)}
    assert keys == set(range(0, 8 * dim, 4))
    halves, n = max(1, dim // 128), 2 if dim == 64 else 4
    values = {L.value_byte(dim, t, h, r, i) for t in range(16) for h in range(halves) for r in range(16) for i in range(n)}
    assert values == set(range(8 * dim))
    for groups in (dim // 32, dim // 64, dim // 128):
        if groups:
            assert {L.plane_word(t, g) for t in range(16) for g in range(groups)} == set(range(0, 64 * groups, 4))
            assert L.record_bytes(dim, groups) == 2 * (8 * dim + 64 * groups) and L.record_bytes(dim, groups) % 128 == 0


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_lane_loads_the_words_of_its_products(dim):
    """Lane (c, g) of a key load: word 4 j + g of token c at position j of its piece; of a value load: tokens 4 g .. 4 g + 3."""
    L = rules()
    for c in range(16):
        for g in range(4):
            for j in range(dim // 32):
                base = c * 32 + g * 8 if dim == 64 else (j // 4) * 1024 + c * 64 + g * 16
                assert L.key_word(dim, c, 4 * j + g) == base + 4 * (j % 4)
            for t in range(4):
                for h in range(max(1, dim // 128)):
                    lane = 16 * g + c
                    want = lane * 8 + 2 * t if dim == 64 else 1024 * h + lane * 16 + 4 * t
                    assert L.value_byte(dim, 4 * g + t, h, c, 0) == want


def test_records_fill_the_cache():
    L = rules()
    seen = {L.record_index(p, 3, h, 64, at) for p in range(5) for h in range(3) for at in range(0, 64, 16)}
    assert seen == set(range(5 * 3 * 4))
    assert L.record_index(2 ** 27 - 1, 1024, 1023, 16, 15) == 2 ** 37 - 1  # past 32 bits


def test_visible_ranges_against_one_key_at_a_time():
    r = random.Random(5)
    L = rules()
    for _ in range(400):
        q, k = r.randint(1, 40), r.choice([0, 1, r.randint(0, 60)])
        causal, window = r.random() < 0.7, r.choice([0, 0, 1, 7, 100, 2 ** 31 - 1])

        def keys(i):
            pos = k - q + i
            return [t for t in range(k) if (not causal or t <= pos) and (not window or t > pos - window)]

        for i in range(q):
            lo, hi = _out(L.visible, 2, i, q, k, int(causal), window)
            assert list(range(lo, hi)) == keys(i), (i, q, k, causal, window)
        union = sorted(set().union(*[keys(i) for i in range(q)]))
        lo, hi = _out(L.request_range, 2, q, k, int(causal), window)
        assert all(lo <= t < hi for t in union)
        if union:
            assert hi == union[-1] + 1
    big = 2 ** 31 - 1
    assert _out(L.visible, 2, 0, 1, big, 1, 0) == (0, big) and _out(L.visible, 2, 0, 1, big, 1, 5) == (big - 5, big)
    assert _out(L.visible, 2, 0, 2 ** 24, 3, 1, 2) == (0, 0)


def test_request_lengths_stay_inside_what_was_checked():
    r = random.Random(6)
    big = [-2 ** 31, -1, 0, 1, 7, 99, 2 ** 31 - 1]
    for _ in range(500):
        n, mq, mk = r.randint(0, 100), r.randint(0, 100), r.randint(0, 1000)
        first, q, k = _out(rules().request, 3, r.choice(big), r.choice(big), r.choice(big), n, mq, mk)
        assert 0 <= first and first + q <= n and 0 <= q <= mq and 0 <= k <= mk


def test_page_plan_counts_new_pages():
    for cached in (0, 1, 15, 16, 17, 31, 32, 33):
        for added in (0, 1, 15, 16, 17, 50):
            before, need = _out(rules().page_plan, 2, cached, added, 4, 100)
            assert before == -(-cached // 16) and before + need == -(-(cached + added) // 16)
    assert _out(rules().page_plan, 2, 2 ** 31 - 1, 2 ** 24, 4, 3) == (3, 0)


def test_shares_cover_every_step():
    for batch, heads, kv in ((1, 1, 1025), (1, 8, 4096), (64, 8, 32768), (1000, 4, 2100), (3, 1, 131072), (2, 8, 5000)):
        for block in (8, 16):
            whole, grid = _out(rules().share, 2, batch, heads, block, kv, 512, kind=C.c_uint32)
            assert not whole and 1 <= grid <= 512
            for keys in (32, 64):
                most = batch * heads * (-(-(kv + keys - 1) // keys) + rules().unit_keys(block) // keys)
                for total in (0, 1, 7, 8, 9, 100, most // 3, most, 2 ** 31 - 1):
                    per, least = rules().share_of(total, grid, keys), 256 // keys
                    assert per % 4 == 0 and per >= least and per * grid >= total
                    assert per == max(least, -(-(-(-total // grid)) // 4) * 4)
                    if grid < 512 and total <= most:  # fewer workgroups than slots: each has its least share
                        assert per == least
    for batch, heads, kv, want in ((5, 2, 0, 1), (5, 2, 1, 1), (5, 2, 1024, 1), (5, 2, 1025, 0), (64, 2, 2048, 1),
                                   (63, 2, 2048, 0), (500, 8, 2049, 0)):
        assert _out(rules().share, 2, batch, heads, 8, kv, 512, kind=C.c_uint32)[0] == want


def test_row_limits():
    """Which requests the decode kernel takes, and in what blocks: by the rows that a kv head's query heads and the new
    tokens make."""
    for batch, query, ratio, kv, want in (
            (1, 1, 4, 9, (64, 8)), (1, 2, 4, 9, (64, 8)), (9, 3, 4, 9, (64, 16)), (1, 16, 4, 9, (64, 16)),
            (1, 17, 4, 10 ** 6, (0, 16)), (2, 17, 4, 30000, (8, 8)), (2, 17, 4, 20000, (0, 16)), (16, 100, 7, 9, (8, 8)),
            (15, 100, 7, 9, (0, 16)), (20, 100, 16, 9, (16, 16)), (20, 100, 17, 9, (0, 16)), (5, 1, 20, 9, (64, 16)),
            (5, 1, 65, 10 ** 6, (0, 16)), (30, 65, 1, 9, (8, 8))):
        assert _out(rules().row_limit, 2, batch, query, ratio, kv, kind=C.c_uint32) == want, (batch, query, ratio)


def test_pieces_cover_a_tile_and_fill_the_gpu():
    r = random.Random(9)
    for _ in range(300):
        keys, pieces = r.randint(1, 200000), r.randint(1, 64)
        each = rules().piece_keys(keys, pieces)
        assert each % 64 == 0 and each >= 256 and each * pieces >= keys
    assert rules().piece_keys(2 ** 31 - 1, 2) * 2 >= 2 ** 31 - 1
    t = rules().tiling
    t.argtypes = [C.c_uint32, C.c_uint32, C.c_uint64, C.c_uint64, C.c_uint32, C.c_uint32, C.c_void_p]
    assert _out(t, 2, 1, 8, 2048 * 4, 2048 * 4, 6144, 256, kind=C.c_uint32) == (64, 1)
    assert _out(t, 2, 1, 1, 300, 300, 100000, 256, kind=C.c_uint32)[1] == 171
    assert _out(t, 2, 1, 1, 300, 300, 300, 256, kind=C.c_uint32)[1] == 2
    assert _out(t, 2, 4, 2, 0, 100, 0, 256, kind=C.c_uint32)[1] == 1


def _geometry(**kw):
    from stark_amd import kv as K
    g = dict(page_count=10, page_size=64, kv_heads=8, head_dim=128, group_size=64)
    g.update(kw)
    return K._Cache(0, 0, *[g[n] for n in ("page_count", "page_size", "kv_heads", "head_dim", "group_size")])


def _size(**kw):
    from stark_amd import qmm as Q
    n = C.c_uint64()
    return Q.lib().stark_qmm_kv_cache_size(C.byref(_geometry(**kw)), C.byref(n)), n.value


def test_cache_size_and_its_refusals():
    from stark_amd import qmm as Q
    assert _size() == (Q.OK, 10 * 64 * 8 * 144)
    assert _size(head_dim=256, group_size=32, page_size=16) == (Q.OK, 10 * 16 * 8 * 2 * (128 + 32))
    assert _size(page_count=2 ** 21, page_size=1024)[0] == Q.INVALID_ARGUMENT
    assert _size(page_count=2 ** 21 - 1, page_size=1024, kv_heads=1024)[1] == (2 ** 21 - 1) * 2 ** 20 * 144
    for bad in (dict(page_size=0), dict(page_size=8), dict(page_size=48), dict(page_size=2048), dict(page_count=0),
                dict(kv_heads=0), dict(kv_heads=1025)):
        assert _size(**bad)[0] == Q.INVALID_ARGUMENT, bad
    assert _size(head_dim=96)[0] == _size(head_dim=512)[0] == Q.UNSUPPORTED
    for bad in (dict(group_size=16), dict(group_size=0), dict(head_dim=64, group_size=128)):
        assert _size(**bad)[0] == Q.UNSUPPORTED_GROUP_SIZE, bad


FAKE = 1 << 20  # an aligned address that no refused call may touch


def _plan(**kw):
    from stark_amd import kv as K
    s = K._PlanArgs()
    for n in ("cached", "added", "free_pages", "free_count", "block_table", "query_start", "kv_lengths", "slots", "positions",
              "free_left", "status"):
        setattr(s, n, FAKE)
    s.struct_size, s.batch, s.token_capacity, s.free_capacity, s.table_stride, s.page_size = C.sizeof(s), 2, 8, 4, 4, 64
    for n, v in kw.items():
        setattr(s, n, v)
    return s


def test_plan_refusals():
    from stark_amd import qmm as Q
    call = Q.lib().stark_qmm_kv_plan
    assert call(None, None) == Q.INVALID_ARGUMENT
    assert call(C.byref(_plan(struct_size=8)), None) == Q.ABI_MISMATCH
    for bad in (dict(page_size=24), dict(page_size=8), dict(batch=2 ** 20 + 1), dict(token_capacity=2 ** 24 + 1),
                dict(free_capacity=2 ** 31), dict(table_stride=2 ** 26), dict(cached=None), dict(added=None),
                dict(free_pages=None), dict(free_count=None), dict(block_table=None), dict(query_start=None),
                dict(kv_lengths=None), dict(slots=None), dict(positions=None), dict(free_left=None), dict(status=None),
                dict(slots=FAKE + 2)):
        assert call(C.byref(_plan(**bad)), None) == Q.INVALID_ARGUMENT, bad


def _cache(**kw):
    g = _geometry(**kw)
    g.data, g.data_size = FAKE, _size(**kw)[1]
    return g


def _append(**kw):
    from stark_amd import kv as K, qmm as Q
    s = K._AppendArgs()
    s.struct_size, s.cache, s.data_type = C.sizeof(s), _cache(), Q.BF16
    s.q = s.q_out = s.k = s.v = s.slots = FAKE
    s.tokens, s.heads = 4, 16
    s.q_token_stride = s.q_out_token_stride = 16 * 128
    s.k_token_stride = s.v_token_stride = 8 * 128
    s.q_head_stride = s.q_out_head_stride = s.k_head_stride = s.v_head_stride = 128
    for n, v in kw.items():
        o = s
        *path, n = n.split("__")
        for x in path:
            o = getattr(o, x)
        setattr(o, n, v)
    return s


def test_append_refusals():
    from stark_amd import qmm as Q
    call = Q.lib().stark_qmm_kv_append
    assert call(None, None) == Q.INVALID_ARGUMENT
    assert call(C.byref(_append(struct_size=1)), None) == Q.ABI_MISMATCH
    assert call(C.byref(_append(data_type=Q.I8)), None) == Q.UNSUPPORTED_DATA_TYPE
    assert call(C.byref(_append(cache__data_size=100)), None) == Q.UNSUPPORTED_LAYOUT
    assert call(C.byref(_append(cache__group_size=48)), None) == Q.UNSUPPORTED_GROUP_SIZE
    assert call(C.byref(_append(tokens=0)), None) == Q.OK
    rot = dict(rotary__rotary_dim=128, rotary__axes=1, rotary__table=FAKE, rotary__positions=FAKE, rotary__table_rows=10)
    for bad in (dict(cache__data=None), dict(cache__data=FAKE + 64), dict(q=None), dict(q_out=None), dict(heads=0), dict(k=None),
                dict(v=None), dict(slots=None), dict(k=FAKE + 1), dict(slots=FAKE + 2), dict(k_head_stride=100),
                dict(k_token_stride=512), dict(v_token_stride=0), dict(q_token_stride=2 ** 41), dict(q_out_head_stride=64),
                dict(tokens=2 ** 24 + 1), dict(rot, rotary__rotary_dim=24), dict(rot, rotary__rotary_dim=144),
                dict(rot, rotary__axes=0), dict(rot, rotary__axes=5), dict(rot, rotary__table=None),
                dict(rot, rotary__table=FAKE + 4), dict(rot, rotary__positions=None), dict(rot, rotary__table_rows=2 ** 31),
                dict(rot, rotary__axes=2, rotary__position_stride=3), dict(q_out=FAKE, q_out_token_stride=17 * 128),
                dict(q_out=FAKE, q_out_head_stride=256, q_out_token_stride=32 * 128)):
        assert call(C.byref(_append(**bad)), None) == Q.INVALID_ARGUMENT, bad
    s = _append(**rot)
    s.rotary.axis_of_pair[63] = 1
    assert call(C.byref(s), None) == Q.INVALID_ARGUMENT


def test_read_refusals():
    from stark_amd import kv as K, qmm as Q
    call = Q.lib().stark_qmm_kv_read

    def args(**kw):
        s = K._ReadArgs()
        s.struct_size, s.cache, s.data_type = C.sizeof(s), _cache(), Q.F32
        s.k = s.v = s.slots = FAKE
        s.tokens, s.k_token_stride, s.v_token_stride, s.k_head_stride, s.v_head_stride = 4, 1024, 1024, 128, 128
        for n, v in kw.items():
            setattr(s, n, v)
        return C.byref(s)

    assert call(None, None) == Q.INVALID_ARGUMENT
    assert call(args(struct_size=2), None) == Q.ABI_MISMATCH
    assert call(args(data_type=Q.U8), None) == Q.UNSUPPORTED_DATA_TYPE
    assert call(args(tokens=0), None) == Q.OK
    for bad in (dict(k=None, v=None), dict(slots=None), dict(k=FAKE + 2), dict(v_token_stride=1000), dict(tokens=2 ** 24 + 1)):
        assert call(args(**bad), None) == Q.INVALID_ARGUMENT, bad


def test_attention_refusals():
    from stark_amd import kv as K, qmm as Q
    call = Q.lib().stark_qmm_kv_attention

    def args(**kw):
        s = K._AttentionArgs()
        s.struct_size, s.cache, s.data_type = C.sizeof(s), _cache(), Q.BF16
        s.q = s.block_table = s.query_start = s.kv_lengths = FAKE
        s.out = FAKE + 2 ** 16
        s.batch, s.tokens, s.heads, s.table_stride, s.max_query, s.max_kv = 2, 4, 16, 8, 2, 512
        s.q_token_stride = s.out_token_stride = 16 * 128
        s.q_head_stride = s.out_head_stride = 128
        s.scale = 0.1
        for n, v in kw.items():
            setattr(s.cache if n == "head_dim" else s, n, v)
        return C.byref(s)

    assert call(None, None) == Q.INVALID_ARGUMENT
    assert Q.lib().stark_qmm_kv_attention_workspace_size(args(), None) == Q.INVALID_ARGUMENT
    assert call(args(struct_size=2), None) == Q.ABI_MISMATCH
    assert call(args(data_type=Q.F32), None) == Q.UNSUPPORTED_DATA_TYPE
    assert call(args(head_dim=80), None) == Q.UNSUPPORTED
    assert call(args(batch=0), None) == call(args(tokens=0), None) == call(args(max_query=0), None) == Q.OK
    for bad in (dict(heads=0), dict(heads=12), dict(heads=65536 + 8), dict(batch=2 ** 20 + 1), dict(tokens=2 ** 24 + 1),
                dict(max_kv=2 ** 31), dict(table_stride=0), dict(table_stride=2 ** 25), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(soft_cap=-1.0), dict(soft_cap=float("nan")), dict(soft_cap=float("inf")),
                dict(q=None), dict(out=None), dict(out=FAKE), dict(block_table=None), dict(query_start=None), dict(kv_lengths=None),
                dict(q=FAKE + 1), dict(lse=FAKE + 2), dict(q_head_stride=64), dict(out_token_stride=128),
                dict(max_kv=2 ** 31 - 1, table_stride=2 ** 25 - 1)):
        assert call(args(**bad), None) == Q.INVALID_ARGUMENT, bad


def test_the_plain_plan_gives_each_token_one_slot():
    """The oracle of the plan's GPU tests, by a property."""
    r = random.Random(7)
    cached, added = [r.randint(0, 70) for _ in range(9)], [r.randint(0, 40) for _ in range(9)]
    table = np.full((9, 16), -1)
    free = list(range(200))
    for b, c in enumerate(cached):
        for i in range(-(-c // 16)):
            table[b, i] = free.pop()
    p = R.plan(cached, added, free, len(free), table, 16, sum(added) + 3)
    used = p["slots"][:sum(added)]
    assert len(set(used)) == sum(added) and (used >= 0).all() and (p["slots"][sum(added):] == -1).all()
    assert p["status"][0] == 0 and list(np.diff(p["query_start"])) == added


def test_a_rotation_table_without_rows_is_refused():
    """A position outside the table gives NaN, but its thread still reads row 0: there has to be one."""
    from stark_amd import qmm as Q
    rot = dict(rotary__rotary_dim=128, rotary__axes=1, rotary__table=FAKE, rotary__positions=FAKE, rotary__table_rows=0)
    assert Q.lib().stark_qmm_kv_append(C.byref(_append(**rot)), None) == Q.INVALID_ARGUMENT


def test_the_workspace_of_a_call_without_rows():
    """No requests, no rows or a bound of none: nothing is launched, so nothing is needed."""
    from stark_amd import kv as K, qmm as Q
    for batch, tokens, most in ((0, 100, 100), (0, 5, 1), (3, 0, 7), (3, 100, 0)):
        s = K._AttentionArgs()
        s.struct_size, s.cache, s.data_type = C.sizeof(s), _geometry(), Q.BF16
        s.batch, s.tokens, s.heads, s.table_stride, s.max_query, s.max_kv = batch, tokens, 8, 64, most, 4096
        n = C.c_uint64(77)
        assert Q.lib().stark_qmm_kv_attention_workspace_size(C.byref(s), C.byref(n)) == Q.OK and n.value == 0


def test_a_read_of_no_tokens():
    """Tensors of no rows have no address."""
    from stark_amd import kv as K, qmm as Q
    s = K._ReadArgs()
    s.struct_size, s.cache, s.data_type = C.sizeof(s), _cache(), Q.F32
    assert Q.lib().stark_qmm_kv_read(C.byref(s), None) == Q.OK


def test_a_plan_whose_outputs_overlap_is_refused():
    """Workgroups read the lengths and the free list while others write."""
    from stark_amd import qmm as Q
    call = Q.lib().stark_qmm_kv_plan
    names = ("cached", "added", "free_pages", "free_count", "block_table", "query_start", "kv_lengths", "slots", "positions",
             "free_left", "status")
    sizes = dict(cached=2, added=2, free_pages=4, free_count=1, block_table=8, query_start=3, kv_lengths=2, slots=8, positions=8,
                 free_left=1, status=1)
    apart = {n: FAKE + 4096 * i for i, n in enumerate(names)}
    outputs = names[4:]
    for o in outputs:
        for n in names:
            if n != o:
                for at in (apart[n], apart[n] + 4 * (sizes[n] - 1), apart[n] - 4 * (sizes[o] - 1)):
                    assert call(C.byref(_plan(**dict(apart, **{o: at}))), None) == Q.INVALID_ARGUMENT, (o, n)
