"""The 4-bit paged key/value cache on the GPU: plan, append, read and attention against their plain 64-bit forms
(tests/kv_ref.py). Rows that the cache stores are compared exactly; attention within the bounds derived there."""
import numpy as np
import pytest
import torch

from tests import kv_ref as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module")
def K(qmm):
    from stark_amd import kv
    return kv


def _dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


def _ints(v):
    return torch.tensor(np.asarray(v, np.int64), dtype=torch.int32).cuda()


def _np(t):
    return t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _same(got, want, label=""):
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{label}: NaN pattern differs"
    bad = (got != want) & ~np.isnan(want)
    assert not bad.any(), f"{label}: {bad.sum()} of {bad.size} differ, first {np.argwhere(bad)[0]}: {got[bad][0]!r} {want[bad][0]!r}"


def _round(x, name):
    """64-bit values as the type holds them (through f32, as the kernels)."""
    with np.errstate(over="ignore"):
        return torch.from_numpy(x).float().to(DT[name]).double().numpy()


# ---------------------------------------------------------------- plan

def _plan_case(rng, batch, page, width, chunk, idle):
    cached = rng.integers(0, page * 3, batch)
    added = np.where(rng.random(batch) < idle, 0, rng.integers(1, chunk + 1, batch))
    have = -(-cached // page)
    width = max(width, int(max(-(-(cached + added) // page)) if batch else 1))
    ids = rng.permutation(int(have.sum()) + int(added.sum()) + 50)
    table = np.full((batch, width), -7)
    at = 0
    for b in range(batch):
        table[b, :have[b]] = ids[at:at + have[b]]
        at += have[b]
    return cached, added, table, ids[at:]


def _run_plan(K, cached, added, free, count, table, page, capacity):
    t = _ints(table)
    op = K.KvPlan(_ints(cached), _ints(added), _ints(free), _ints([count]), t, page, capacity)
    for n in ("query_start", "kv_lengths", "slots", "positions", "free_left", "status"):
        getattr(op, n).fill_(-99)
    op.encode()
    op.encode()  # a second pass over the same lengths writes the same
    torch.cuda.synchronize()
    want = R.plan(cached, added, free, count, np.asarray(table), page, capacity)
    for n, w in want.items():
        got = t if n == "block_table" else getattr(op, n)
        _same(_np(got).astype(np.int64), w, n)
    return op


@pytest.mark.parametrize("batch,page,chunk,idle", [(1, 16, 1, 0.0), (8, 64, 1, 0.3), (5, 16, 40, 0.0), (255, 32, 9, 0.2),
                                                   (256, 16, 3, 0.5), (257, 128, 200, 0.1), (700, 16, 5, 0.9), (3, 1024, 3000, 0), (1024, 16, 2, 0.5),
                                                   (1025, 32, 3, 0.2), (2300, 16, 1, 0.6)])
def test_plan(K, batch, page, chunk, idle):
    cached, added, table, free = _plan_case(np.random.default_rng(batch), batch, page, 4, chunk, idle)
    _run_plan(K, cached, added, free, len(free), table, page, int(added.sum()) + 5)


def test_plan_flags(K):
    rng = np.random.default_rng(3)
    cached, added, table, free = _plan_case(rng, 40, 16, 4, 30, 0.1)
    total = int(added.sum())
    op = _run_plan(K, cached, added, free, 7, table, 16, total)
    assert _np(op.status)[0] == K.OUT_OF_PAGES and _np(op.free_left)[0] == 0
    _run_plan(K, cached, added, free, 0, table, 16, total)
    op = _run_plan(K, cached, added, free, len(free) + 100, table, 16, total - 20)  # a count past the list is cut
    assert _np(op.status)[0] & K.TOO_MANY_TOKENS
    bad = cached.copy()
    bad[3], bad[4] = -5, 0
    table[3:5] = -1
    op = _run_plan(K, bad, added, free, len(free), table, 16, total)
    assert _np(op.status)[0] == K.BAD_LENGTH


def test_plan_table_full_and_no_requests(K):
    cached, added = np.array([30, 0]), np.array([40, 3])
    table = np.array([[5, 6, -1], [-1, -1, -1]])
    op = _run_plan(K, cached, added, np.arange(20) + 30, 20, table, 16, 43)
    assert _np(op.status)[0] == K.TABLE_FULL
    op = K.KvPlan(_ints([]), _ints([]), _ints([4]), _ints([1]), torch.zeros(0, 3, dtype=torch.int32, device="cuda"), 16, 2)
    op.encode()
    torch.cuda.synchronize()
    assert _np(op.slots).tolist() == [-1, -1] and _np(op.query_start).tolist() == [0] and _np(op.free_left).tolist() == [1]


# ---------------------------------------------------------------- append and read

def _table(rows, pairs):
    a = np.arange(rows)[:, None] * 10000.0 ** (-np.arange(pairs) / pairs)
    return np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)


def _strided(x, dtype, how):
    """The rows as a view with the given strides: dense, one of a fused q/k/v row, heads outside tokens, or unaligned."""
    t = _dev(x, dtype)
    if how == "fused":
        wide = torch.full((t.shape[0], 2 * t.shape[1] + 1, t.shape[2]), 3.0, dtype=dtype, device="cuda")
        wide[:, 1:1 + t.shape[1]] = t
        return wide[:, 1:1 + t.shape[1]]
    if how == "heads":
        return t.transpose(0, 1).contiguous().transpose(0, 1)
    if how == "odd":
        wide = torch.full((t.shape[0] * (t.shape[1] * t.shape[2] + 3) + 1,), 3.0, dtype=dtype, device="cuda")
        v = wide[1:].view(t.shape[0], -1)[:, :t.shape[1] * t.shape[2]].unflatten(1, t.shape[1:])
        v.copy_(t)
        return v
    return t


APPEND = [
    # dim, group, kv heads, query heads, tokens, page, type, axes (0: no rotation), rotary dims, interleaved, strides
    (128, 64, 2, 8, 1, 16, "bf16", 1, 128, False, "dense"),
    (128, 32, 3, 3, 37, 64, "bf16", 3, 128, False, "fused"),
    (128, 128, 1, 7, 130, 32, "f16", 0, 0, False, "heads"),
    (64, 32, 4, 4, 50, 16, "f32", 1, 32, False, "odd"),
    (64, 64, 2, 6, 19, 16, "bf16", 2, 64, True, "dense"),
    (256, 64, 2, 2, 33, 128, "f16", 1, 192, True, "odd"),
    (256, 32, 1, 4, 21, 16, "bf16", 4, 256, False, "dense"),
    (256, 128, 2, 2, 5, 1024, "f32", 0, 0, False, "dense"),
    (128, 64, 1, 0, 70, 16, "f32", 1, 16, False, "fused"),
]


@pytest.mark.parametrize("dim,group,kvh,heads,tokens,page,dtype,axes,rd,inter,how", APPEND)
def test_append_and_read(K, dim, group, kvh, heads, tokens, page, dtype, axes, rd, inter, how):
    rng = np.random.default_rng(dim + group + tokens)
    q, k, v = (_round(rng.normal(0, 2, (tokens, h, dim)), dtype) for h in (max(heads, 1), kvh, kvh))
    k += 0
    pages = -(-tokens // page) + 2
    slots = rng.permutation(pages * page)[:tokens]
    cache = K.KvCache(pages, page, kvh, dim, group)
    cache.data.fill_(0xA5)
    rot = None
    wq, wk = q, k
    if axes:
        table = _table(97, rd // 2)
        positions = rng.integers(0, 97, (axes, tokens))
        pick = rng.integers(0, axes, rd // 2)
        wide = _ints(np.concatenate([positions, np.full((axes, 3), 2 ** 31 - 1)], 1))
        rot = K.Rotary(_dev(table), wide[:, :tokens] if axes > 1 else wide[0], pick, inter)
        wq, wk = R.rotate(q, table, positions, pick, inter), R.rotate(k, table, positions, pick, inter)
    dq, dk, dv = (_strided(x, DT[dtype], how) for x in (q, k, v))
    q_out = torch.full_like(_strided(q, DT[dtype], "dense"), 7.0)
    op = K.KvAppend(cache, dk, dv, _ints(slots), *((dq, q_out) if heads else ()), rotary=rot)
    op.encode()
    outs = [_strided(np.zeros((tokens, kvh, dim)), DT["f32"], how) for _ in range(2)]
    K.KvRead(cache, _ints(slots), *outs).encode()
    torch.cuda.synchronize()
    want = [R.stored(wk, group), R.stored(v, group)]
    for got, w, n in zip(outs, want, "kv"):
        _same(_np(got), _round(w, "f32"), n)
    if heads:
        # products and sum in f32 (2^-24 of each), then the type's own rounding; without a rotation the values as they are
        near = 2.0 ** -23 * 2 * np.abs(q).max(-1, keepdims=True)

        def same_q(got, label):
            if not axes:
                return _same(got, q, label)
            assert (np.abs(got - wq) <= near + R.EPS[dtype] * (np.abs(wq) + near) + 2.0 ** -25).all(), label
            if rd < dim:
                _same(got[..., rd:], q[..., rd:], label)

        same_q(_np(q_out), "q")
        if how != "heads":
            K.KvAppend(cache, dk, dv, _ints(slots), dq, dq, rotary=rot).encode()  # in place
            torch.cuda.synchronize()
            same_q(_np(dq), "q in place")
    for name in DT:
        one = torch.zeros(tokens, kvh, dim, dtype=DT[name], device="cuda")
        K.KvRead(cache, _ints(slots), None, one).encode()
        torch.cuda.synchronize()
        _same(_np(one), _round(want[1], name), f"v as {name}")


def test_rotated_keys_close_to_a_tie_of_their_planes(K):
    """Enough rotated groups that some have a minimum or a range within f32's rounding of half way between two f16
    values, where one rounding and two differ."""
    rng = np.random.default_rng(0)
    t, kvh, dim = 4096, 8, 128
    k = _round(rng.normal(0, 1, (t, kvh, dim)) + rng.normal(0, 2, (1, kvh, dim)), "bf16")
    table, positions = _table(300, 64), rng.integers(0, 300, (1, t))
    cache = K.KvCache(t // 64, 64, kvh, dim, 64)
    slots, dk = _ints(np.arange(t)), _dev(k, torch.bfloat16)
    K.KvAppend(cache, dk, dk, slots, rotary=K.Rotary(_dev(table), _ints(positions[0]))).encode()
    out = torch.zeros(t, kvh, dim, device="cuda")
    K.KvRead(cache, slots, out, None).encode()
    torch.cuda.synchronize()
    turned = R.rotate(k, table, positions, [0] * 64, False)
    low = turned.reshape(t, kvh, 2, 64).min(-1)
    with np.errstate(all="ignore"):
        assert (low.astype(np.float16) != low.astype(np.float32).astype(np.float16)).any()
    _same(_np(out), _round(R.stored(turned, 64), "f32"), "k")


@pytest.mark.parametrize("dim,group", [(64, 32), (128, 64), (256, 128)])
def test_groups_at_the_edges(K, dim, group):
    """Constant groups, zeros of both signs, subnormals, values half way between codes, the largest values, and groups
    that the format does not hold."""
    rows = []

    def add(f):
        x = np.zeros(dim)
        x[:group] = f
        x[group:] = np.linspace(-1, 1, dim - group)
        rows.append(x)

    i = np.arange(group)
    add(0.0 * i)
    add(np.where(i % 2, 0.0, -0.0))
    add(0.0 * i + 3.3)
    add(2.0 ** -40 * i)
    add(2.0 ** -24 * (i % 16))
    add((i % 31) / 2.0)          # scale 1: every second value is half way
    add(-(i % 31) / 2.0 + 0.25)
    add(np.where(i == 3, 32768.0, -32768.0))
    add(np.where(i == 3, 32770.0, 1.0))
    add(np.where(i == 5, np.nan, i))
    add(np.where(i == 6, np.inf, i))
    add(np.where(i == 7, -np.inf, i))
    add(1000.0 + i * 2.0 ** -10)  # a range below a step of its bias
    x = _round(np.array(rows)[:, None, :], "f32")
    n = x.shape[0]
    cache = K.KvCache(2, 16, 1, dim, group)
    slots = _ints(np.arange(n) + 5)
    K.KvAppend(cache, _dev(x, torch.float32), _dev(x, torch.float32), slots).encode()
    k, v = torch.zeros(n, 1, dim, device="cuda"), torch.zeros(n, 1, dim, device="cuda")
    K.KvRead(cache, slots, k, v).encode()
    torch.cuda.synchronize()
    want = _round(R.stored(x, group), "f32")
    _same(_np(k), want, "k")
    _same(_np(v), want, "v")


@pytest.mark.parametrize("dim,dtype,inter,axes,shift", [(64, "bf16", False, 3, 0), (128, "f16", True, 1, 2), (64, "f32", False, 1, 0)])
def test_an_append_of_many_rows_is_its_parts(K, dim, dtype, inter, axes, shift):
    """Several rows to a thread (a large call) and one (small ones) leave the same cache and the same queries."""
    rng = np.random.default_rng(dim + axes)
    tokens, heads, kvh, page, group = 6001, 41, 5, 64, 32
    q, k, v = (_round(rng.normal(0, 1, (tokens, n, dim)), dtype) for n in (heads, kvh, kvh))
    q, k, v = (_dev(x, DT[dtype]) for x in (q, k, v))
    flat = torch.zeros(500 * dim + shift, device="cuda")  # shift: rows of the table that are not 16-byte aligned
    table = flat[shift:].view(500, dim // 2, 2)
    table.copy_(_dev(_table(500, dim // 2), torch.float32))
    positions = _ints(rng.integers(0, 500, (axes, tokens)))
    pick = np.sort(rng.integers(0, axes, dim // 2))
    slots = _ints(rng.permutation(100 * page)[:tokens])
    caches, outs = [], []
    for step in (tokens, 37):
        cache, out = K.KvCache(100, page, kvh, dim, group), q.clone()
        for a in range(0, tokens, step):
            part = slice(a, a + step)
            K.KvAppend(cache, k[part], v[part], slots[part], out[part], out[part],
                       K.Rotary(table, positions[:, part], pick, inter)).encode()
        caches.append(cache.data), outs.append(out)
    torch.cuda.synchronize()
    assert torch.equal(*caches) and torch.equal(outs[0].view(torch.uint8), outs[1].view(torch.uint8))


def test_slots_outside_the_cache_write_and_read_nothing(K):
    rng = np.random.default_rng(1)
    cache = K.KvCache(3, 16, 2, 64, 32)
    cache.data.copy_(torch.from_numpy(rng.integers(0, 256, cache.data.numel()).astype(np.uint8)))
    before = cache.data.clone()
    slots = _ints([-1, 48, 49, 2 ** 31 - 1, -2 ** 31, -48])
    k = _dev(rng.normal(0, 1, (6, 2, 64)), torch.bfloat16)
    q = _dev(rng.normal(0, 1, (6, 4, 64)), torch.bfloat16)
    q_out = torch.zeros_like(q)
    K.KvAppend(cache, k, k, slots, q, q_out).encode()
    torch.cuda.synchronize()
    assert torch.equal(cache.data, before) and torch.equal(q, q_out)
    out = torch.full((6, 2, 64), 5.0, device="cuda")
    K.KvRead(cache, slots, out, out.clone()).encode()
    torch.cuda.synchronize()
    assert (out == 5.0).all()
    # one row changes its own bytes only: each row's codes and planes are 2 heads x 2 x (32 + 8) bytes
    K.KvAppend(cache, k[:1], k[:1], _ints([17])).encode()
    torch.cuda.synchronize()
    assert 0 < int((cache.data != before).sum()) <= 2 * 2 * (32 + 8)


def test_positions_outside_the_table_give_nan(K):
    cache = K.KvCache(1, 16, 1, 64, 32)
    x = torch.ones(4, 1, 64, device="cuda")
    q_out = torch.empty_like(x)
    rot = K.Rotary(_dev(_table(10, 16)), _ints([9, 10, -1, 0]))
    K.KvAppend(cache, x, x, _ints([0, 1, 2, 3]), x, q_out, rot).encode()
    torch.cuda.synchronize()
    nan = torch.isnan(q_out)
    assert not nan[0].any() and not nan[3].any()
    assert nan[1, 0, :32].all() and nan[2, 0, :32].all() and not nan[1:3, 0, 32:].any()


# ---------------------------------------------------------------- attention

class Served:
    """Requests in a paged cache of random page order: q rows, and keys and values as the cache holds them."""

    def __init__(self, K, seed, requests, heads, kvh, dim, group, page, dtype, pad_tokens=0, how="dense", width=None,
                 edit=None):
        rng = np.random.default_rng(seed)
        self.K, self.requests, self.kvh, self.dim, self.dtype = K, requests, kvh, dim, dtype
        need = [-(-kv // page) for _, kv in requests]
        pages = sum(need) + 1
        order = rng.permutation(pages)
        self.cache = K.KvCache(pages, page, kvh, dim, group)
        # what no request owns is noise: NaN planes among it
        self.cache.data.copy_(torch.from_numpy(rng.integers(0, 256, self.cache.data.numel()).astype(np.uint8)))
        table = np.full((len(requests), max(max(need), width or 1)), -1)
        slots, at = [], 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            t = np.arange(requests[b][1])
            slots.append(table[b, t // page] * page + t % page)
            at += n
        total = sum(kv for _, kv in requests)
        k = rng.normal(0, 1, (total, kvh, dim)) * np.exp(rng.normal(0, 0.5, (1, kvh, dim))) + rng.normal(0, 1, (1, kvh, dim))
        v = rng.normal(0, 1, (total, kvh, dim)) + rng.normal(0, 0.5, (1, kvh, dim))
        if edit:
            edit(k, v)
        flat = _ints(np.concatenate(slots) if slots else [])
        self.slots = slots
        self.k, self.v = torch.zeros(total, kvh, dim, device="cuda"), torch.zeros(total, kvh, dim, device="cuda")
        if total:
            K.KvAppend(self.cache, _dev(k, torch.float32), _dev(v, torch.float32), flat).encode()
            K.KvRead(self.cache, flat, self.k, self.v).encode()
        tokens = sum(q for q, _ in requests) + pad_tokens
        self.q = _strided(_round(rng.normal(0, 1, (tokens, heads, dim)), dtype), DT[dtype], how)
        self.table = _ints(table)
        self.query_start = _ints(np.concatenate([[0], np.cumsum([q for q, _ in requests])]))
        self.kv_lengths = _ints([kv for _, kv in requests])
        self.max_query, self.max_kv = max(q for q, _ in requests), max(kv for _, kv in requests)
        self.out = _strided(np.full((tokens, heads, dim), 9.0), DT[dtype], how)
        self.lse = torch.full((tokens, heads), 9.0, device="cuda")

    def operator(self, **kw):
        if not kw.pop("with_lse", True):
            self.lse = None
        kw.setdefault("max_query", self.max_query)
        kw.setdefault("max_kv", self.max_kv)
        return self.K.KvAttention(self.cache, self.q, self.out, self.table, self.query_start, self.kv_lengths,
                                  lse=self.lse, **kw)

    def check(self, causal=True, window=0, soft_cap=0.0, scale=None, hidden=None):
        """hidden: request -> keys whose page is not in the cache."""
        q, k, v, out = _np(self.q), _np(self.k), _np(self.v), _np(self.out)
        lse = None if self.lse is None else _np(self.lse)
        each, at, kat = q.shape[1] // self.kvh, 0, 0
        wide = 0 if self.max_query * each <= 64 else 2 if lse is None and self.dtype == "bf16" else 1
        scale = self.dim ** -0.5 if scale is None else scale
        for b, (n, kv) in enumerate(self.requests):
            for h in range(self.kvh):
                rows = q[at:at + n, h * each:(h + 1) * each]
                want, wl, tol, dl = R.attention(rows, k[kat:kat + kv, h], v[kat:kat + kv, h], scale, causal, window,
                                                soft_cap, wide)
                got = out[at:at + n, h * each:(h + 1) * each]
                label = f"request {b} ({n} rows, {kv} keys) head {h}"
                assert np.array_equal(np.isnan(got), np.isnan(want)), f"{label}: NaN pattern"
                ok = ~np.isnan(want)
                err = np.abs(got - want)[ok]
                # a rounding to f16 below its normal range is off by 2^-25
                bound = tol[ok] * 1.001 + R.EPS[self.dtype] * (np.abs(want[ok]) + tol[ok]) + 2.0 ** -25
                assert (err <= bound).all(), f"{label}: off by {err.max()} (bound there {bound[np.argmax(err - bound)]})"
                dead = np.isneginf(wl)
                assert (got[dead] == 0).all()
                if lse is None:
                    continue
                gl = lse[at:at + n, h * each:(h + 1) * each]
                assert np.array_equal(np.isneginf(gl), dead), f"{label}: empty rows"
                fin = ~dead & np.isfinite(wl)
                assert (np.abs(gl[fin] - wl[fin]) <= dl[fin] + 2.0 ** -23 * np.abs(wl[fin])).all(), f"{label}: lse"
            at, kat = at + n, kat + kv
        assert (out[at:] == 9.0).all() and (lse is None or (lse[at:] == 9.0).all()), "rows behind the last request"


ATTEND = [
    # requests (query rows, keys), heads, kv heads, dim, group, page, type, options
    ([(1, 1)], 4, 4, 128, 64, 16, "bf16", {}),
    ([(1, 17)], 8, 2, 128, 64, 16, "bf16", {}),
    ([(1, 300), (1, 31), (1, 33), (1, 1000)], 8, 2, 128, 64, 64, "bf16", {}),
    ([(1, 5000)], 8, 1, 128, 32, 64, "f16", {}),
    ([(1, 700), (1, 64)], 7, 1, 128, 128, 16, "f16", {}),
    ([(1, 513), (1, 2)], 20, 1, 64, 32, 32, "bf16", {}),
    ([(1, 259)], 2, 2, 64, 64, 128, "f16", {}),
    ([(1, 800)], 4, 2, 256, 64, 16, "bf16", {}),
    ([(1, 65), (3, 66)], 2, 1, 256, 32, 32, "f16", {}),
    ([(1, 129)], 16, 2, 256, 128, 1024, "bf16", {}),
    ([(1, 0), (0, 5), (1, 9), (0, 0)], 4, 2, 128, 64, 16, "bf16", {}),
    ([(5, 900), (3, 40), (1, 900), (4, 4)], 32, 4, 128, 32, 16, "bf16", {}),
    ([(7, 3)], 4, 2, 128, 64, 16, "bf16", {}),                       # rows before the first key see nothing
    ([(5, 2), (3, 3)], 4, 4, 64, 32, 16, "f16", dict(causal=False)),
    ([(33, 33), (1, 100), (70, 200)], 8, 2, 128, 64, 32, "bf16", {}),
    ([(130, 130)], 4, 1, 64, 32, 16, "f16", {}),
    ([(40, 500), (257, 300)], 4, 2, 128, 64, 64, "bf16", dict(window=50)),
    ([(1, 500), (2, 77)], 4, 2, 128, 64, 64, "f16", dict(window=1)),
    ([(1, 4000)], 4, 1, 128, 64, 16, "bf16", dict(window=1000)),
    ([(1, 300), (40, 90)], 4, 2, 128, 64, 16, "bf16", dict(soft_cap=5.0)),
    ([(2, 300), (65, 90)], 8, 2, 64, 64, 16, "f16", dict(soft_cap=30.0, window=64)),
    ([(20, 450)], 4, 2, 128, 64, 16, "bf16", dict(causal=False)),
    ([(20, 450)], 4, 2, 128, 64, 16, "bf16", dict(causal=False, window=60)),
    ([(100, 260), (1, 33)], 4, 2, 256, 64, 16, "bf16", {}),
    ([(50, 600)], 4, 2, 128, 32, 16, "f16", dict(scale=0.5)),
    ([(300, 2100), (200, 200), (1, 900)], 8, 2, 128, 64, 64, "bf16", {}),
    ([(64, 1700)], 6, 1, 256, 32, 32, "f16", {}),
    ([(90, 1300)], 5, 1, 64, 64, 64, "bf16", dict(window=700)),
    ([(48, 48)], 40, 2, 128, 128, 16, "bf16", {}),
    ([(40, 60), (70, 70)], 4, 2, 64, 32, 16, "bf16", {}),
    ([(200, 333)], 2, 2, 64, 64, 32, "bf16", dict(soft_cap=8.0)),
    ([(80, 100)], 8, 4, 128, 32, 16, "bf16", dict(scale=-0.3)),
    ([(50, 77), (1, 5)], 8, 4, 128, 64, 16, "bf16", dict(scale=0.0)),
    ([(2, 77)], 8, 4, 128, 64, 16, "bf16", dict(scale=-0.2)),
    ([(90, 200)], 2, 1, 256, 128, 16, "bf16", {}),
    ([(3, 100)] * 70 + [(1, 30)] * 3, 4, 2, 64, 32, 16, "bf16", {}),   # more requests than lanes
    ([(1, 600)] * 300, 2, 1, 64, 64, 16, "f16", {}),
    # lengths whose steps workgroups share, in blocks of 8 and of 16 rows
    ([(1, 30)] * 70 + [(1, 2100), (2, 40)], 4, 2, 64, 32, 16, "bf16", {}),
    ([(1, 1100), (0, 3), (1, 2500), (1, 90)], 8, 2, 128, 64, 64, "bf16", {}),
    ([(5, 1400), (3, 1100), (1, 0)], 32, 4, 128, 32, 16, "f16", {}),
    ([(1, 1700), (2, 1200)], 4, 1, 256, 32, 32, "bf16", dict(soft_cap=20.0)),
    ([(1, 1900), (1, 1300)], 20, 1, 64, 64, 16, "bf16", dict(window=1200)),
]


@pytest.mark.parametrize("requests,heads,kvh,dim,group,page,dtype,options", ATTEND)
def test_attention(K, requests, heads, kvh, dim, group, page, dtype, options):
    s = Served(K, len(requests) + heads + dim, requests, heads, kvh, dim, group, page, dtype, pad_tokens=3)
    s.operator(**options).encode()
    torch.cuda.synchronize()
    s.check(**options)


@pytest.mark.parametrize("requests,heads,kvh,dim,group,page,dtype,options", [
    c for c in ATTEND if c[6] == "bf16"])
def test_attention_without_lse(K, requests, heads, kvh, dim, group, page, dtype, options):
    """bf16 outputs alone: prompts round the keys to f16."""
    s = Served(K, len(requests) + heads + dim, requests, heads, kvh, dim, group, page, dtype, pad_tokens=3)
    s.operator(with_lse=False, **options).encode()
    torch.cuda.synchronize()
    s.check(**options)


@pytest.mark.parametrize("how", ["fused", "heads", "odd"])
def test_attention_strides(K, how):
    s = Served(K, 4, [(1, 70), (2, 300), (40, 90)], 6, 3, 128, 64, 16, "bf16", how=how, pad_tokens=1)
    s.operator().encode()
    torch.cuda.synchronize()
    s.check()


def test_attention_wider_bounds_and_table(K):
    """Bounds and a block table larger than any request: the split into chunks is by the bounds."""
    s = Served(K, 8, [(1, 70), (2, 300), (3, 20)], 8, 2, 128, 64, 16, "bf16", width=700)
    s.operator(max_query=5, max_kv=11000).encode()
    torch.cuda.synchronize()
    s.check()


def _nan_at(tokens, dims):
    def edit(k, v):
        for x in (k, v):
            x[tokens, :, dims] = np.nan
    return edit


@pytest.mark.parametrize("rows", [6, 70])
def test_nan_keys_reach_only_rows_that_see_them(K, rows):
    """Keys and values that are not numbers behind a row's position, or before its window: every earlier row is as if
    they were not there."""
    kv = rows + 140
    s = Served(K, 2, [(rows, kv)], 4, 2, 128, 64, 16, "bf16", edit=_nan_at(kv - 3, 5))
    s.operator().encode()
    torch.cuda.synchronize()
    s.check()
    out = _np(s.out)
    assert not np.isnan(out[:rows - 3]).any() and np.isnan(out[rows - 3:]).all()

    def only_values(k, v):
        v[kv - 3, :, 70] = np.inf

    s = Served(K, 3, [(rows, kv)], 4, 2, 128, 64, 16, "bf16", edit=only_values)
    s.operator().encode()
    torch.cuda.synchronize()
    s.check()
    out = _np(s.out)
    assert not np.isnan(out[:rows - 3]).any() and np.isnan(out[rows - 3:, :, 64:]).all()
    assert not np.isnan(out[:, :, :64]).any()
    s = Served(K, 4, [(rows, kv)], 4, 2, 128, 64, 16, "bf16", edit=_nan_at(2, 5))
    s.operator(window=20).encode()
    torch.cuda.synchronize()
    s.check(window=20)
    assert not np.isnan(_np(s.out)).any()


@pytest.mark.parametrize("with_lse", [True, False])
@pytest.mark.parametrize("rows,group", [(2, 64), (70, 64), (70, 32), (70, 128)])
def test_scores_that_rise_along_the_keys(K, rows, group, with_lse):
    """Scores that grow (or fall, by the sign of a row's sum) by some 60 binary orders: the running reference of the
    exponents has to move several times."""
    def ramp(k, v):
        k += np.linspace(0, 40, len(k))[:, None, None]

    s = Served(K, 29, [(rows, 900)], 4, 2, 128, group, 64, "bf16", edit=ramp)
    s.operator(with_lse=with_lse).encode()
    torch.cuda.synchronize()
    s.check()


@pytest.mark.parametrize("rows", [1, 40])
def test_value_scales_far_apart(K, rows):
    """Values of the first keys near zero and later ones large (and the other way round): the power of two on the
    probabilities is not the first keys' alone."""
    for first, later in ((1e-6, 1.0), (1e-4, 3000.0), (2000.0, 1e-3), (0.0, 500.0)):
        def edit(k, v):
            v[:64] *= first
            v[64:] *= later
        s = Served(K, 6, [(rows, 900)], 4, 1, 128, 64, 16, "f16", edit=edit)
        s.operator().encode()
        torch.cuda.synchronize()
        s.check()


@pytest.mark.parametrize("rows", [1, 40])
def test_query_magnitudes(K, rows):
    """Rows of q of all zeros, tiny and large values, and an infinity (NaN in its row only)."""
    s = Served(K, 7, [(rows, 200)], 8, 2, 128, 64, 16, "bf16")
    s.q[0, 0] = 0
    s.q[0, 1] *= 2.0 ** -100
    s.q[0, 2] *= 2.0 ** 6
    s.q[rows - 1, 7, 3] = float("inf")
    s.operator().encode()
    torch.cuda.synchronize()
    out = _np(s.out)
    assert np.isnan(out[rows - 1, 7]).all() and np.isnan(out).sum() == 128
    s.q[rows - 1, 7, 3] = 0
    s.operator().encode()
    torch.cuda.synchronize()
    s.check()


@pytest.mark.parametrize("rows", [1, 40])
def test_page_ids_outside_the_cache_hide_their_keys(K, rows):
    s = Served(K, 9, [(rows, 200), (rows, 90)], 4, 2, 128, 64, 16, "bf16")
    keep = [t for t in range(200) if not 32 <= t < 48 and not 64 <= t < 80]
    table = s.table.clone()
    s.table[0, 2], s.table[0, 4] = -1, s.cache.page_count
    s.operator(causal=False).encode()
    torch.cuda.synchronize()
    # as without those keys
    q, k, v, out = _np(s.q), _np(s.k), _np(s.v), _np(s.out)
    for h in range(2):
        want, _, tol, _ = R.attention(q[:rows, 2 * h:2 * h + 2], k[:200][keep][:, h], v[:200][keep][:, h], 128 ** -0.5, False, 0,
                                      0.0, 1 if rows > 1 else 0)
        got = out[:rows, 2 * h:2 * h + 2]
        assert (np.abs(got - want) <= tol + R.EPS["bf16"] * (np.abs(want) + tol)).all()
    s.table[0, :13] = -5
    s.operator().encode()
    torch.cuda.synchronize()
    assert (_np(s.out)[:rows] == 0).all() and np.isneginf(_np(s.lse)[:rows]).all()
    s.table.copy_(table)
    s.operator().encode()
    torch.cuda.synchronize()
    s.check()


def test_device_lengths_past_the_bounds_are_cut(K):
    """query_start and kv_lengths that say more than the bounds and the table: nothing outside is read or written."""
    s = Served(K, 5, [(2, 60), (1, 50)], 4, 2, 128, 64, 16, "bf16", pad_tokens=2)
    s.query_start.copy_(_ints([0, 2, 2 ** 31 - 1]))
    s.kv_lengths.copy_(_ints([60, 2 ** 31 - 1]))
    s.operator(max_query=2).encode()
    torch.cuda.synchronize()
    assert (_np(s.out)[4:] == 9.0).all()
    s.query_start.copy_(_ints([-4, -2, 5]))
    s.kv_lengths.copy_(_ints([-1, 50]))
    s.operator().encode()
    torch.cuda.synchronize()


# ---------------------------------------------------------------- together, as a serving loop calls them

def _serve_loop(K, steps, capture, stream):
    """Requests that start at unlike lengths, grow by the added tokens of each step, and attend after each append.
    Every step is checked against rows kept in 64 bits."""
    rng = np.random.default_rng(11)
    batch, page, kvh, heads, dim, group = 3, 16, 2, 8, 128, 64
    width, cap = 20, 48
    cache = K.KvCache(80, page, kvh, dim, group)
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    cached, added = torch.zeros(batch, dtype=torch.int32, device="cuda"), torch.zeros(batch, dtype=torch.int32, device="cuda")
    free, free_count = _ints(rng.permutation(80)), _ints([80])
    plan = K.KvPlan(cached, added, free, free_count, table, page, cap)
    rope = _table(400, dim // 2)
    q, k, v = (torch.zeros(cap, h, dim, dtype=torch.bfloat16, device="cuda") for h in (heads, kvh, kvh))
    out = torch.zeros_like(q)
    append = K.KvAppend(cache, k, v, plan.slots, q, q, K.Rotary(_dev(rope), plan.positions))
    attend = K.KvAttention(cache, q, out, table, plan.query_start, plan.kv_lengths, max_query=40, max_kv=width * page)

    def step():
        plan.encode()
        append.encode()
        attend.encode()

    graph = None
    if capture:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    lengths = np.zeros(batch, int)
    rows_k, rows_v = ([np.zeros((0, kvh, dim)) for _ in range(batch)] for _ in range(2))
    for a in steps:
        cached.copy_(_ints(lengths))
        added.copy_(_ints(a))
        host = [_round(rng.normal(0, 1, (cap, h, dim)), "bf16") for h in (heads, kvh, kvh)]
        for t, x in zip((q, k, v), host):
            t.copy_(_dev(x, torch.bfloat16))
        out.fill_(9.0)
        torch.cuda.synchronize()
        if graph:
            graph.replay()
        else:
            with torch.cuda.stream(stream):
                step()
        torch.cuda.synchronize()
        assert _np(plan.status)[0] == 0
        free_count.copy_(plan.free_left)
        at = 0
        got = _np(out)
        for b in range(batch):
            n = a[b]
            pos = lengths[b] + np.arange(n)
            rk = R.rotate(host[1][at:at + n], rope, pos[None], [0] * 64, False)
            rq = _round(R.rotate(host[0][at:at + n], rope, pos[None], [0] * 64, False), "bf16")
            rows_k[b] = np.concatenate([rows_k[b], R.stored(rk, group)])
            rows_v[b] = np.concatenate([rows_v[b], R.stored(host[2][at:at + n], group)])
            lengths[b] += n
            for h in range(kvh):
                want, _, tol, _ = R.attention(rq[:, 4 * h:4 * h + 4], rows_k[b][:, h], rows_v[b][:, h], dim ** -0.5, True, 0,
                                              0.0, 2)
                err = np.abs(got[at:at + n, 4 * h:4 * h + 4] - want)
                assert (err <= tol + R.EPS["bf16"] * (np.abs(want) + tol)).all(), (b, n, lengths[b], err.max())
            at += n
        assert (got[at:] == 9.0).all()


STEPS = [[30, 1, 0], [1, 1, 17], [1, 1, 1], [0, 0, 0], [1, 0, 33], [16, 15, 1], [1, 1, 1]]


def test_a_serving_loop(K):
    _serve_loop(K, STEPS, False, torch.cuda.current_stream())


def test_a_serving_loop_on_another_stream(K):
    _serve_loop(K, STEPS, False, torch.cuda.Stream())


def test_a_serving_loop_as_a_replayed_graph(K):
    _serve_loop(K, STEPS, True, torch.cuda.Stream())


def test_two_streams_at_once(K):
    """Two operators with workspaces of their own, their calls in flight together, give what each gives alone."""
    many = [Served(K, 20 + i, [(1, 6000), (1, 4000 + i)], 8, 2, 128, 64, 16, "bf16") for i in range(2)]
    ops = [s.operator() for s in many]
    assert all(o.workspace_bytes for o in ops)
    streams = [torch.cuda.Stream() for _ in many]
    torch.cuda.synchronize()
    for _ in range(20):
        for o, s in zip(ops, streams):
            o.encode(s)
    torch.cuda.synchronize()
    for s in many:
        s.check()


def test_results_do_not_depend_on_the_run(K):
    s = Served(K, 30, [(1, 9000), (4, 700), (100, 500)], 8, 2, 128, 64, 16, "bf16")
    op = s.operator()
    seen = set()
    for _ in range(4):
        s.out.fill_(9.0)
        op.encode()
        torch.cuda.synchronize()
        seen.add(s.out.view(torch.int16).cpu().numpy().tobytes())
    assert len(seen) == 1


def test_a_cache_past_32_bits(K):
    """Records beyond 2^32 bytes and slots near the end of the cache."""
    pages = 5 * 2 ** 30 // (64 * 8 * 144) + 1
    cache = K.KvCache(pages, 64, 8, 128, 64)
    assert cache.data.numel() > 5 * 2 ** 30
    rng = np.random.default_rng(2)
    t = 100
    slots = np.concatenate([(pages - 1) * 64 + np.arange(64), (pages - 2) * 64 + np.arange(36)])
    k, v = _round(rng.normal(0, 1, (t, 8, 128)), "bf16"), _round(rng.normal(0, 1, (t, 8, 128)), "bf16")
    K.KvAppend(cache, _dev(k, torch.bfloat16), _dev(v, torch.bfloat16), _ints(slots)).encode()
    q = _round(rng.normal(0, 1, (1, 8, 128)), "bf16")
    out = torch.zeros(1, 8, 128, dtype=torch.bfloat16, device="cuda")
    K.KvAttention(cache, _dev(q, torch.bfloat16), out, _ints([[pages - 1, pages - 2]]), _ints([0, 1]), _ints([t]), 1, t).encode()
    torch.cuda.synchronize()
    sk, sv = R.stored(k, 64), R.stored(v, 64)
    for h in range(8):
        want, _, tol, _ = R.attention(q[:, h:h + 1], sk[:, h], sv[:, h], 128 ** -0.5, True, 0, 0.0, 0)
        err = np.abs(_np(out)[:, h:h + 1] - want)
        assert (err <= tol + R.EPS["bf16"] * (np.abs(want) + tol)).all(), (h, err.max())


def test_refusals(K, qmm):
    cache = K.KvCache(4, 16, 2, 128, 64)
    q = torch.zeros(2, 4, 128, dtype=torch.bfloat16, device="cuda")
    table, start, lens = _ints([[0, 1]]), _ints([0, 2]), _ints([20])

    def refused(f, status=qmm.INVALID_ARGUMENT):
        with pytest.raises(qmm.MatmulError) as e:
            f()
        assert e.value.status == status

    def attention(**kw):
        a = dict(cache=cache, q=q, out=torch.empty_like(q), block_table=table, query_start=start, kv_lengths=lens, max_query=2,
                 max_kv=32)
        a.update(kw)
        return K.KvAttention(**a)

    attention().encode()
    refused(lambda: attention(q=q.float(), out=q.float()), qmm.UNSUPPORTED_DATA_TYPE)
    refused(lambda: attention(out=q.half()))
    refused(lambda: attention(q=q[:, :3], out=q[:, :3].clone()))
    refused(lambda: attention(kv_lengths=lens.long()))
    refused(lambda: attention(query_start=start[:1]))
    refused(lambda: attention(lse=torch.zeros(3, device="cuda")))
    refused(lambda: attention(soft_cap=-2.0))
    refused(lambda: attention(q=q.transpose(1, 2).contiguous().transpose(1, 2)))
    wide = _ints([list(range(4)) * 500])
    need = attention(block_table=wide, max_kv=20000)
    assert need.workspace_bytes
    refused(lambda: attention(block_table=wide, max_kv=20000, workspace=need.workspace[:-16]).encode(), qmm.WORKSPACE_TOO_SMALL)
    refused(lambda: K.KvAppend(cache, q, q, _ints([0, 1])))
    refused(lambda: K.KvAppend(cache, q[:, :2], q[:, :2].half(), _ints([0, 1])))
    refused(lambda: K.KvAppend(cache, q[:, :2], q[:, :2], _ints([0])))
    refused(lambda: K.KvAppend(cache, q[:, :2], q[:, :2], _ints([0, 1]), q))
    refused(lambda: K.KvRead(cache, _ints([0, 1]), None, None))
    refused(lambda: K.KvCache(4, 16, 2, 96, 32), qmm.UNSUPPORTED)
    with pytest.raises(ValueError):
        K.KvAppend(cache, q[:, :2].cpu(), q[:, :2], _ints([0, 1]))
