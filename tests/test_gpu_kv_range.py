"""The 4-bit cache's operators at the ends of what they accept: magnitudes of queries, scores, values and soft caps, rows
behind a window that nothing wrote, and calls that both attention kernels share."""
import numpy as np
import pytest
import torch

from tests import kv_ref as R
from tests.test_gpu_kv import DT, Served, _dev, _ints, _np, _round, _same, _strided, _table

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(qmm):
    from stark_amd import kv
    return kv


def _run(s, **kw):
    op = s.operator(**kw)
    op.encode()
    torch.cuda.synchronize()
    return op


def _requests(s):
    """Of each request and key head: its rows' slice of the call, the query heads, q, k, v (64 bits)."""
    q, k, v = _np(s.q), _np(s.k), _np(s.v)
    each, at, kat = q.shape[1] // s.kvh, 0, 0
    for n, kv in s.requests:
        for h in range(s.kvh):
            heads = slice(h * each, (h + 1) * each)
            yield slice(at, at + n), heads, q[at:at + n, heads], k[kat:kat + kv, h], v[kat:kat + kv, h]
        at, kat = at + n, kat + kv


def _one_key_wins(s, scale, wide):
    """Scores so far apart that the softmax is 1 at one key and 0 at all others. The winner's probability times its
    value's scale is one rounding to f16 (2^-11 of that part, beside at most twice the largest value), with `wide` the
    value another, then the output's own. The score: f32 products and sums of dim terms (kv_ref), f32 lse."""
    out = _np(s.out)
    lse = None if s.lse is None else _np(s.lse)
    for rows, heads, q, k, v in _requests(s):
        n, each, dim = q.shape
        reach = 2 * np.abs(k).max()
        for h in range(each):
            x = q[:, h] @ k.T * scale
            mag = abs(scale) * (np.abs(q[:, h]) @ np.abs(k.T) + np.abs(q[:, h]).sum(-1, keepdims=True) * reach)
            x = np.where(np.arange(len(k)) <= len(k) - n + np.arange(n)[:, None], x, -np.inf)
            win = x.argmax(-1)
            top = x.max(-1)
            error = (mag * ((dim + 16) * 2.0 ** -24 + (2.0 ** -11 if wide == 2 else 0.0))).max(-1)
            second = np.where(np.arange(len(k)) == win[:, None], -np.inf, x).max(-1)
            assert (top - second > 2 * error + 100).all(), "the inputs leave more than one key"
            want = v[win]
            # (|s c| <= |v| + |b|, and |b| at most the row's largest value)
            tol = (2.0 ** -11 + (2.0 ** -11 if wide else 0.0) + 2.0 ** -20) * (np.abs(want) + np.abs(want).max(-1, keepdims=True))
            got = out[rows, heads][:, h]
            assert np.isfinite(got).all(), f"head {h}: not finite in rows {np.argwhere(~np.isfinite(got).all(-1)).ravel()}"
            assert (np.abs(got - want) <= tol + R.EPS[s.dtype] * (np.abs(want) + tol) + 2.0 ** -25).all(), f"head {h}"
            if lse is not None:
                gl = lse[rows, heads][:, h]
                assert (np.abs(gl - top) <= error + 2.0 ** -21 * np.abs(top)).all(), f"lse of head {h}"


@pytest.mark.parametrize("with_lse", [True, False])
@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("power,one_sign", [(100, False), (118, False), (121, False), (122, True)])
def test_queries_near_the_end_of_bf16(K, rows, power, one_sign, with_lse):
    """Finite scores of queries of 2^power, where the power of two that brings them to f16 meets the scale. One sign: the
    sum of a row's values passes f32, its scores do not."""
    def edit(k, v):
        k[:] = np.where(np.arange(128) % 2, 1.0, -1.0) * (1.0 if one_sign else np.sign(k)) * 0.25
        k[7] += 1.0

    s = Served(K, 41, [(rows, 300)], 4, 2, 128, 64, 16, "bf16", edit=edit)
    x = torch.ones_like(s.q) if one_sign else torch.where(s.q > 0, 1.0, 1.25)
    s.q.copy_((x + torch.arange(rows, device="cuda").view(-1, 1, 1) / 128).to(torch.bfloat16) * 2.0 ** power)
    _run(s, with_lse=with_lse)
    _one_key_wins(s, 128 ** -0.5, 0 if rows == 2 else 1 if with_lse else 2)


@pytest.mark.parametrize("rows", [2, 40])
def test_tiny_queries_with_a_large_scale(K, rows):
    """Queries of 2^-76 under a scale of 2^64 and more: scores of ordinary size."""
    s = Served(K, 42, [(rows, 200)], 4, 2, 128, 64, 16, "bf16")
    s.q.mul_(2.0 ** -66)
    _run(s, scale=2.0 ** 63)
    s.check(scale=2.0 ** 63)


@pytest.mark.parametrize("with_lse", [True, False])
@pytest.mark.parametrize("rows,dtype", [(2, "bf16"), (2, "f16"), (40, "bf16"), (40, "f16")])
@pytest.mark.parametrize("size", [200.0, 2400.0, 3000.0, 3413.0, 5000.0, 20000.0])
def test_scores_past_the_whole_numbers_of_f32(K, rows, dtype, size, with_lse):
    """Scores of 2^20 to 2^33, whose neighbours in f32 are up to 512 apart: one key wins by far, and what a sum of two
    roundings leaves must not count as a probability of 2^64."""
    if dtype == "f16" and not with_lse:
        return
    sign = np.where(np.random.default_rng(3).random(128) < 0.5, -1.0, 1.0)

    def edit(k, v):
        k[:] = 0.1 * size * np.sign(k)
        k[61] = size * sign
        v[:] = np.clip(8.0 * v, -11.0, 11.0)  # scales of 22 / 15

    s = Served(K, 43, [(rows, 300)], 4, 2, 128, 64, 16, dtype, edit=edit)
    x = _dev(sign, torch.float32) * (1 + torch.arange(rows, device="cuda").view(-1, 1, 1) / 64)
    x = x * (1 + torch.arange(4, device="cuda").view(1, -1, 1) / 8)
    s.q.copy_((x * size).to(DT[dtype]))
    _run(s, with_lse=with_lse)
    _one_key_wins(s, 128 ** -0.5, 0 if rows == 2 else 1 if with_lse else 2)


@pytest.mark.parametrize("with_lse", [True, False])
@pytest.mark.parametrize("rows", [2, 40])
def test_rows_of_nothing_but_very_low_scores(K, rows, with_lse):
    """Scores of -1e31 and below are scores: the row is not an empty one."""
    def edit(k, v):
        k[:] = -1.0
        k[5] = -0.25

    s = Served(K, 44, [(rows, 90)], 4, 2, 128, 64, 16, "bf16", edit=edit)
    s.q.copy_(torch.ones_like(s.q) * (1 + torch.arange(rows, device="cuda").view(-1, 1, 1) / 64) * 2.0 ** 108)
    _run(s, with_lse=with_lse)
    _one_key_wins(s, 128 ** -0.5, 0 if rows == 2 else 1 if with_lse else 2)


@pytest.mark.parametrize("with_lse", [True, False])
@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("cap", [0.5, 30.0, 1e3, 1e5, 2.0 ** 20])
def test_soft_caps(K, rows, cap, with_lse):
    """A large cap leaves small scores as they are. The bound is kv_ref's with the cap's own error, 2^-20 of it there, put
    at 2^-20 of the largest score: cap tanh(s / cap) is never larger than s, and no term of it is."""
    s = Served(K, 45, [(rows, 300)], 4, 2, 128, 64, 16, "bf16")
    _run(s, soft_cap=cap, with_lse=with_lse)
    out, wide = _np(s.out), 0 if rows == 2 else 1 if with_lse else 2
    for rs, heads, q, k, v in _requests(s):
        want, wl, tol, dl = R.attention(q, k, v, 128 ** -0.5, True, 0, cap, wide)
        top = np.abs(np.einsum("nhd,td->nht", q, k) * 128 ** -0.5).max(-1)
        less = 2.0 ** -20 * cap - 2.0 ** -20 * np.minimum(top, cap)  # [n, heads]
        tol = tol - 2 * less[..., None] * np.abs(v).max(0)
        err = np.abs(out[rs, heads] - want)
        assert (err <= tol * 1.001 + R.EPS["bf16"] * (np.abs(want) + tol)).all(), (err / tol).max()
        if with_lse:
            assert (np.abs(_np(s.lse)[rs, heads] - wl) <= dl - less + 2.0 ** -23 * np.abs(wl)).all()


def _small_values(s, wide):
    """As Served.check for outputs in bf16, without its 2^-25 of f16 outputs."""
    out = _np(s.out)
    for rows, heads, q, k, v in _requests(s):
        k, v = k[-s.window:], v[-s.window:]  # (0: all; a window is for one row)
        want, _, tol, _ = R.attention(q, k, v, 128 ** -0.5, True, 0, 0.0, wide)
        got = out[rows, heads]
        err = np.abs(got - want)
        assert (err <= tol * 1.001 + R.EPS["bf16"] * (np.abs(want) + tol)).all(), (err / np.abs(want)).max()


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("first,later", [(0.0, 1e-5), (0.0, 1e-4), (0.0, 1.0), (0.0, 3000.0), (1e-5, 1e-5)])
@pytest.mark.parametrize("keys", [129, 140, 900])
def test_zeros_before_small_values(K, rows, first, later, keys):
    """Value groups of zeros have a scale of 0, which says nothing of the scales behind them."""
    def edit(k, v):
        k *= 0.1  # near-equal weights
        v[:128] *= first
        v[128:] *= later

    s = Served(K, 46, [(rows, keys)], 8, 2, 128, 64, 16, "bf16", edit=edit)
    s.window = 0
    _run(s)
    _small_values(s, 0 if rows == 1 else 1)


def test_values_before_the_window_do_not_set_the_scale(K):
    """Large values of keys that a window leaves behind, in the step where it begins."""
    def edit(k, v):
        k *= 0.1
        v[:] *= 1e-5
        v[512:543] = np.sign(v[512:543]) * 30000.0

    s = Served(K, 47, [(1, 546)], 8, 2, 128, 64, 16, "bf16", edit=edit)
    s.window = 546 - 543
    _run(s, window=s.window)
    _small_values(s, 0)


@pytest.mark.parametrize("dtype,with_lse", [("bf16", True), ("bf16", False), ("f16", True)])
@pytest.mark.parametrize("rows", [2, 40])
def test_a_first_key_above_all_others(K, rows, dtype, with_lse):
    """An attention sink: a key 15 above the rest (in natural logarithms) whose value is zero, so that the output is what
    the other keys' small probabilities make. An error d of the scores moves it by 2 d sum w |v - out|; a probability is
    held to 2^-12 of itself (2^-11 in kv_ref's bound), or below f16's normal range to 2^-33 of the largest."""
    def edit(k, v):
        k[:, :, 1:] *= 0.2
        k[:, :, 0] = 0.0
        k[0], v[0] = 0.0, 0.0
        k[0, :, 0] = 16.0

    s = Served(K, 48, [(rows, 100)], 4, 2, 128, 64, 16, dtype, edit=edit)
    s.q[:, :, 0] = 10.625
    _run(s, with_lse=with_lse)
    out, wide = _np(s.out), 0 if rows == 2 else 1 if with_lse else 2
    for rs, heads, q, k, v in _requests(s):
        n = q.shape[0]
        seen = np.arange(len(k)) <= len(k) - n + np.arange(n)[:, None]
        for h in range(q.shape[1]):
            x = np.where(seen, q[:, h] @ k.T * 128 ** -0.5, -np.inf)
            mag = 128 ** -0.5 * (np.abs(q[:, h]) @ np.abs(k.T) + np.abs(q[:, h]).sum(-1, keepdims=True) * 2 *
                                 np.abs(k).max(-1))
            w = np.exp(x - x.max(-1, keepdims=True))
            total = w.sum(-1, keepdims=True)
            w /= total
            want = w @ v
            d = np.where(seen, 144 * 2.0 ** -24 * mag + (2.0 ** -11 * mag if wide == 2 else 0.0) + 2.0 ** -22 * 40, 0.0)
            a = w @ (np.abs(v) + np.abs(v).max(-1, keepdims=True))
            tol = np.einsum("nt,ntd->nd", 2 * w * d, np.abs(v - want[:, None])) + a * (2.0 ** -11 + (2.0 ** -10 if wide else 0)
                                                                                       + 2.0 ** -18)
            tol += 2.0 ** -33 * (np.abs(v).sum(0) + np.abs(v).max(-1).sum())
            err = np.abs(out[rs, heads][:, h] - want)
            own = 2.0 ** -25 if dtype == "f16" else 0.0  # of outputs below f16's normal range
            assert (err <= tol + R.EPS[dtype] * (np.abs(want) + tol) + own).all(), (err / tol).max()


@pytest.mark.parametrize("dtype,with_lse", [("bf16", True), ("bf16", False), ("f16", True)])
@pytest.mark.parametrize("rows", [1, 40])
def test_unwritten_rows_before_the_window(K, rows, dtype, with_lse):
    """Pages that lie wholly before every row's window may have been given away: what they hold, finite planes whose
    values pass f16 here, reaches nothing."""
    n = 500
    s = Served(K, 49, [(rows, n)], 4, 2, 128, 64, 16, dtype)
    window = n - rows + 1 - 432  # the first row's window begins in the fourth page of a tile of 64 keys
    assert s.table.shape[1] == 32 and window > 0
    used = set(_np(s.table).ravel().tolist())
    spare = next(p for p in range(s.cache.page_count) if p not in used)
    page = s.cache.data.view(s.cache.page_count, -1)
    page[spare] = 0x7B
    s.table[0, :432 // 16] = spare
    _run(s, window=window, with_lse=with_lse)
    s.check(window=window)


def test_f32_queries_that_nearly_cancel(K):
    """A rotated f32 value is rounded once: what is left of a difference of nearly equal products is as exact as any."""
    rng = np.random.default_rng(50)
    t, heads, dim = 64, 4, 128
    table, positions = _table(300, 64), rng.integers(1, 300, (1, t))
    q = rng.normal(0, 1, (t, heads, dim))
    c, s = (table[positions[0], :, i].astype(np.float64)[:, None] for i in (0, 1))
    q[:, ::2, :64] = q[:, ::2, 64:] * s / np.where(np.abs(c) > 1e-3, c, 1.0)     # first halves go to about 0
    q[:, 1::2, 64:] = -q[:, 1::2, :64] * s / np.where(np.abs(c) > 1e-3, c, 1.0)  # second halves do
    q = _round(q, "f32")
    for inter in (False, True):
        rows = q if not inter else q.reshape(t, heads, 2, 64).swapaxes(2, 3).reshape(t, heads, dim)
        cache, out = K.KvCache(4, 16, 1, dim, 64), torch.zeros(t, heads, dim, device="cuda")
        k = torch.zeros(t, 1, dim, device="cuda")
        K.KvAppend(cache, k, k, _ints(np.arange(t)), _dev(rows, torch.float32), out,
                   K.Rotary(_dev(table), _ints(positions[0]), interleaved=inter)).encode()
        torch.cuda.synchronize()
        want = R.rotate(rows, table, positions, [0] * 64, inter)
        assert (np.abs(want) < 1e-6).mean() > 0.2
        # one rounding of the exact products' sum to 64 bits, and one to f32
        size = np.abs(rows).max()
        assert (np.abs(_np(out) - want) <= 2.0 ** -24 * np.abs(want) + 2.0 ** -51 * size + 2.0 ** -149).all()


@pytest.mark.parametrize("requests,heads,kvh,dim,group,page,dtype,options", [
    ([(1, 40)] * 150 + [(300, 500)] + [(1, 70)] * 100, 8, 2, 64, 32, 16, "bf16", {}),
    ([(600, 700)] + [(0, 3)] * 70 + [(1, 33)] * 130, 4, 2, 128, 64, 16, "f16", {}),
    ([(1, 20)] * 64 + [(2, 9)] + [(129, 140)] * 2, 16, 8, 64, 64, 16, "bf16", dict(window=30)),
])
def test_few_long_requests_among_many_short_ones(K, requests, heads, kvh, dim, group, page, dtype, options):
    """Workgroups by the rows that the call has: each request's are found by its place, in batches of more than 64."""
    s = Served(K, 51, requests, heads, kvh, dim, group, page, dtype, pad_tokens=3)
    _run(s, **options)
    s.check(**options)


def test_thousands_of_requests_with_a_long_bound(K):
    """4096 requests, any of which could be 16384 rows long: one row tile each and head would be 2^24 workgroups."""
    rng = np.random.default_rng(52)
    batch, long, heads, kvh, dim = 4096, 300, 32, 8, 64
    cache = K.KvCache(20, 16, kvh, dim, 32)
    k, v = (_dev(rng.normal(0, 1, (320, kvh, dim)), torch.float32) for _ in range(2))
    K.KvAppend(cache, k, v, _ints(np.arange(320))).encode()
    K.KvRead(cache, _ints(np.arange(320)), k, v).encode()
    rows = batch - 1 + long
    q = torch.zeros(16384, heads, dim, dtype=torch.bfloat16, device="cuda")
    q[:rows] = _dev(rng.normal(0, 1, (rows, heads, dim)), torch.bfloat16)
    out = torch.full_like(q, 9.0)
    table = np.zeros((batch, 20))
    table[-1] = np.arange(20)
    start = np.append(np.arange(batch), rows)
    op = K.KvAttention(cache, q, out, _ints(table), _ints(start), _ints([7] * (batch - 1) + [long]), max_query=16384, max_kv=320)
    op.encode()
    torch.cuda.synchronize()
    assert (out[rows:] == 9.0).all()
    hq, hk, hv, ho = _np(q[:rows]), _np(k), _np(v), _np(out[:rows])
    for h in range(kvh):
        mine = slice(4 * h, 4 * h + 4)
        for part, n, causal in ((slice(0, batch - 1), 7, False), (slice(batch - 1, rows), long, True)):
            want, _, tol, _ = R.attention(hq[part, mine], hk[:n, h], hv[:n, h], dim ** -0.5, causal, 0, 0.0, 2)
            assert (np.abs(ho[part, mine] - want) <= tol + R.EPS["bf16"] * (np.abs(want) + tol)).all()


SHARED = [
    # decode rows in blocks of 8 or 16 whose steps workgroups share, and prompts in pieces: one workspace for both
    ([(1, 2500)] * 15 + [(100, 3000)], 8, 2, 128, 64, 64, "bf16", {}),
    ([(1, 2100), (2, 2300), (3, 40)] * 6 + [(150, 2200), (0, 7)], 12, 2, 64, 32, 16, "f16", dict(window=1500)),
    ([(70, 2600)] + [(1, 2200)] * 16 + [(90, 100)], 32, 2, 128, 128, 32, "bf16", {}),
    ([(1, 2100)] * 16 + [(40, 2100)], 14, 1, 256, 64, 64, "bf16", dict(soft_cap=20.0)),
    ([(1, 16000), (60, 9000), (1, 20000), (1, 3)], 4, 2, 64, 64, 64, "bf16", {}),
    # each unit a workgroup of its own, beside prompts
    ([(1, 900)] * 17 + [(30, 900)], 10, 1, 256, 32, 32, "f16", {}),
    ([(1, 64), (5, 64), (1, 0), (33, 200)] * 8, 6, 3, 64, 32, 16, "bf16", dict(causal=False)),
    # blocks of 16 rows of wide heads
    ([(1, 300), (2, 1500), (4, 90)], 16, 1, 256, 128, 64, "bf16", {}),
    ([(3, 700)], 16, 2, 256, 32, 16, "f16", dict(window=300)),
    ([(5, 1300), (5, 2000), (2, 10)], 12, 1, 256, 64, 32, "bf16", dict(soft_cap=12.0)),
]


@pytest.mark.parametrize("with_lse", [True, False])
@pytest.mark.parametrize("requests,heads,kvh,dim,group,page,dtype,options", SHARED)
def test_decode_rows_and_prompts_in_one_call(K, requests, heads, kvh, dim, group, page, dtype, options, with_lse):
    s = Served(K, 53, requests, heads, kvh, dim, group, page, dtype, pad_tokens=2)
    _run(s, with_lse=with_lse, **options)
    s.check(**options)


def test_decode_rows_and_prompts_in_one_captured_call(K):
    """The combined call captured, replayed over other lengths within its bounds, and against the eager call each time."""
    s = Served(K, 54, [(1, 2500)] * 17 + [(90, 2600)], 8, 2, 128, 64, 64, "bf16", pad_tokens=2)
    op = s.operator()
    op.encode()
    torch.cuda.synchronize()
    s.check()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        op.encode()
    lengths, start = s.kv_lengths.clone(), s.query_start.clone()
    for i, cut in enumerate((0, 700, 2000, 2400, 0)):
        s.kv_lengths.copy_(lengths - cut)
        s.query_start.copy_(start)
        if i % 2:
            s.query_start[-1] = 17 + 40  # a shorter prompt
        s.out.fill_(9.0), s.lse.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        got = s.out.clone(), s.lse.clone()
        s.out.fill_(9.0), s.lse.fill_(9.0)
        op.encode()
        torch.cuda.synchronize()
        assert torch.equal(got[0].view(torch.int16), s.out.view(torch.int16)) and torch.equal(got[1], s.lse)
    s.check()


@pytest.mark.parametrize("heads,kvh,cut", [(4, 2, 2), (60, 2, 5)])
def test_lengths_past_the_bounds_give_the_rows_that_are_left(K, heads, kvh, cut):
    """query_start below 0 and past the rows, a negative length and one past the bound: what kv::request leaves of each
    request is computed, and every other row stays as it was."""
    s = Served(K, 55, [(2, 60), (9, 50)], heads, kvh, 64, 32, 16, "bf16", pad_tokens=2)
    q, k, v = _np(s.q), _np(s.k), _np(s.v)
    for start, lengths, rows, keys in (([0, 2, 2 ** 31 - 1], [60, 2 ** 31 - 1], [(0, 2), (2, cut)], [60, 60]),
                                       ([-4, -2, 5], [-1, 50], [(0, 0), (0, cut)], [0, 50])):
        s.query_start.copy_(_ints(start))
        s.kv_lengths.copy_(_ints(lengths))
        s.out.fill_(9.0), s.lse.fill_(9.0)
        _run(s, max_query=cut)
        out, lse = _np(s.out), _np(s.lse)
        left = np.ones(q.shape[0], bool)
        for b, ((at, n), kv) in enumerate(zip(rows, keys)):
            left[at:at + n] = False
            if kv > s.requests[b][1]:
                continue  # keys that nothing wrote: what these rows are is not said
            kk, vv = (x[:kv] if b == 0 else x[60:60 + kv] for x in (k, v))
            for h in range(kvh if n else 0):
                each = heads // kvh
                mine = slice(h * each, (h + 1) * each)
                want, wl, tol, dl = R.attention(q[at:at + n, mine], kk[:, h], vv[:, h], 64 ** -0.5, True, 0, 0.0,
                                                1 if cut * each > 64 else 0)
                assert (np.abs(out[at:at + n, mine] - want) <= tol + R.EPS["bf16"] * (np.abs(want) + tol)).all()
                assert (np.abs(lse[at:at + n, mine] - wl) <= dl + 2.0 ** -23 * np.abs(wl)).all()
        assert (out[left] == 9.0).all() and (lse[left] == 9.0).all()


@pytest.mark.parametrize("requests,heads,kvh", [([(1, 70), (2, 300), (1, 9)], 8, 2), ([(1, 70)] * 70 + [(100, 300)], 8, 2),
                                                ([(60, 300), (130, 200)], 4, 2), ([(1, 2100)] * 30 + [(90, 2200)], 8, 2)])
def test_rows_ahead_of_the_first_request(K, requests, heads, kvh):
    """query_start may begin behind row 0: the rows before it are no request's."""
    s = Served(K, 56, requests, heads, kvh, 128, 64, 16, "bf16", pad_tokens=300)
    s.query_start += 290
    s.q = torch.roll(s.q, 290, 0)
    _run(s)
    s.q, s.out, s.lse = (torch.roll(t, -290, 0) for t in (s.q, s.out, s.lse))
    s.check()


def test_two_rows_for_one_slot(K):
    """What the slot holds is of the two: each group has one row's scale and bias, and codes of either. No other slot
    changes."""
    rng = np.random.default_rng(57)
    t, kvh, dim, group = 64, 2, 128, 32
    x = _round(rng.normal(0, 1, (2 * t, kvh, dim)) + rng.normal(0, 3, (2 * t, 1, 1)), "bf16")
    cache = K.KvCache(t // 16 + 1, 16, kvh, dim, group)
    cache.data.fill_(0xA5)
    slots = _ints(np.concatenate([np.arange(t), rng.permutation(t)]))
    dev = _dev(x, torch.bfloat16)
    K.KvAppend(cache, dev, dev, slots).encode()
    out = [torch.zeros(t, kvh, dim, device="cuda") for _ in range(2)]
    K.KvRead(cache, _ints(np.arange(t)), *out).encode()
    torch.cuda.synchronize()
    assert (cache.data.view(t // 16 + 1, -1)[-1] == 0xA5).all()
    order = _np(slots)
    sums = [p.astype(np.float64)[..., None] for p in R.planes(x, group)]
    for got in out:
        g = _np(got).reshape(t, kvh, dim // group, group)
        fits = np.zeros(g.shape[:-1], bool)
        for rows in (np.arange(t), t + np.argsort(order[t:])):
            scale, bias = (p[rows] for p in sums)
            code = (g - bias) / scale
            fits |= ((np.abs(code - np.rint(code)) < 1e-3) & (code > -0.5) & (code < 15.5)).all(-1)
        assert fits.all()


def test_the_workspace_is_that_of_the_tensors_device(K, monkeypatch):
    """Its size depends on the device's compute units: the query is made with that device current."""
    s = Served(K, 58, [(1, 5000)], 8, 2, 128, 64, 16, "bf16")
    seen, inner = [], torch.cuda.device

    class Spy(inner):
        def __enter__(self):
            seen.append(self.idx)
            return super().__enter__()

    monkeypatch.setattr(torch.cuda, "device", Spy)
    op = s.operator()
    assert op.workspace_bytes and s.q.device.index in seen


@pytest.mark.parametrize("requests,heads,kvh,dim,group,options", [
    ([(1, 3000), (3, 5000), (1, 40)], 8, 1, 128, 32, {}),
    ([(1, 20000)], 8, 2, 64, 64, {}),
    ([(5, 700), (2, 1500)], 8, 1, 256, 64, dict(soft_cap=30.0)),
    ([(70, 2500), (30, 900)], 8, 2, 128, 64, {}),
    ([(200, 1200)], 4, 2, 64, 32, dict(window=700)),
    ([(90, 6000)], 4, 1, 256, 128, {}),
    ([(1, 900)] * 17 + [(60, 3000)], 8, 2, 128, 128, {}),
])
def test_f16_outputs_are_off_by_their_own_rounding(K, requests, heads, kvh, dim, group, options):
    """Over all rows of a call, as root mean square: the error of a correctly rounded output, and 5 % for all else. That is
    products of probabilities and values to 2^-22 of each and sums in f32, two orders below f16's 2^-12; a probability or a
    value held in one f16 alone would make it 30 % and more."""
    def edit(k, v):
        k *= 0.5
        v -= v.mean(0)  # outputs as small as the keys' average leaves them: its parts' errors show

    s = Served(K, 60, requests, heads, kvh, dim, group, 16, "f16", edit=edit)
    _run(s, **options)
    out, got, best = _np(s.out), 0.0, 0.0
    for rows, mine, q, k, v in _requests(s):
        want = R.attention(q, k, v, dim ** -0.5, True, options.get("window", 0), options.get("soft_cap", 0.0), 0)[0]
        got += ((out[rows, mine] - want) ** 2).sum()
        best += ((want.astype(np.float16).astype(np.float64) - want) ** 2).sum()
    assert got <= 1.05 ** 2 * best, (got / best) ** 0.5


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,dim,group", [(1, 128, 32), (2, 64, 64), (3, 256, 128), (20, 128, 32), (40, 64, 64)])
def test_lse_is_as_exact_as_f32_sums(K, rows, dim, group, dtype):
    """With one key the lse is the score. A dozen f32 roundings (sums of each scale group, planes) of terms of some two times
    a score's size, beside the seven or so of a plain sum in f32: within 8 times that sum's error, as root mean square."""
    batch = 64
    s = Served(K, 61, [(rows, 1)] * batch, 16, 2, dim, group, 16, dtype)
    _run(s, causal=False)
    lse, ours, plain = _np(s.lse), 0.0, 0.0
    q32, k32 = s.q.float(), s.k
    for i, (at, mine, q, k, v) in enumerate(_requests(s)):
        b, h = divmod(i, 2)
        want = np.einsum("nhd,d->nh", q, k[0]) * dim ** -0.5
        f32 = _np((q32[at, mine] * k32[b, h]).sum(-1) * dim ** -0.5)
        ours += ((lse[at, mine] - want) ** 2).sum()
        plain += ((f32 - want) ** 2).sum()
    assert ours <= 64 * plain, (ours / plain) ** 0.5


@pytest.mark.parametrize("rows,dim,group", [(6, 128, 32), (70, 128, 64), (70, 64, 64), (70, 256, 32)])
def test_values_that_are_no_numbers_in_f16_calls(K, rows, dim, group):
    """They reach the rows that see them, in their scale group and no other value."""
    kv, bad = rows + 140, dim - 3

    def edit(k, v):
        v[kv - 3, :, bad] = np.inf

    s = Served(K, 62, [(rows, kv)], 4, 2, dim, group, 16, "f16", edit=edit)
    _run(s)
    s.check()
    nan = np.isnan(_np(s.out))
    at = bad // group * group
    assert nan[rows - 3:, :, at:at + group].all() and nan.sum() == 3 * 4 * group


@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("size", [2.0 ** -24, 2.0 ** -20, 2.0 ** -17, 2.0 ** -14, 3000.0])
def test_value_scales_at_both_ends_in_f16_calls(K, rows, size):
    """Scales that are f16 subnormals, and the largest: the stored values are exact multiples, and so are the operands that
    the kernels make of them. Outputs below f16's normal range are off by half its least step."""
    def edit(k, v):
        v[:] = np.clip(v, -2.5, 2.5) / 2.5 * 8 * size

    s = Served(K, 63, [(rows, 200)], 4, 2, 128, 64, 16, "f16", edit=edit)
    _run(s)
    s.check()
    out = _np(s.out)
    for rs, mine, q, k, v in _requests(s):
        want, _, tol, _ = R.attention(q, k, v, 128 ** -0.5, True, 0, 0.0, 0)
        assert (np.abs(out[rs, mine] - want) <= tol + R.EPS["f16"] * (np.abs(want) + tol) + 2.0 ** -25).all()
