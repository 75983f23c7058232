"""Plain 64-bit forms of the 4-bit key/value cache's operators (numpy), written from their definitions, and the
bounds that the kernels' arithmetic stays within."""
import numpy as np

LIMIT = 32768.0
EPS = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}  # half a step, relative


def planes(x, group):
    """f16 scales and biases [.., groups] of 64-bit rows, NaN where a group does not fit."""
    g = x.reshape(x.shape[:-1] + (x.shape[-1] // group, group))
    with np.errstate(all="ignore"):
        bad = ~np.all(np.abs(g) <= LIMIT, axis=-1)
        lo, hi = g.min(-1), g.max(-1)
        s = ((hi - lo) / 15.0).astype(np.float32).astype(np.float16)
        b = lo.astype(np.float32).astype(np.float16)
    return np.where(bad, np.float16(np.nan), s), np.where(bad, np.float16(np.nan), b)


def stored(x, group):
    """What the cache holds of 64-bit rows, as 64-bit values."""
    s, b = (p.astype(np.float64)[..., None] for p in planes(x, group))
    g = x.reshape(x.shape[:-1] + (x.shape[-1] // group, group))
    with np.errstate(all="ignore"):
        q = np.where(s > 0, np.clip(np.rint((g - b) / np.where(s > 0, s, 1.0)), 0, 15), 0.0)
        return (q * s + b).reshape(x.shape)


def rotate(x, table, positions, axes, interleaved):
    """64-bit rows [tokens, heads, dim] turned by f32 (cos, sin) rows; positions [axes, tokens]."""
    y = x.copy()
    pairs = table.shape[1]
    for i in range(pairs):
        p = positions[axes[i]]
        inside = (p >= 0) & (p < table.shape[0])
        cs = np.where(inside[:, None], table[np.where(inside, p, 0), i].astype(np.float64), np.nan)
        c, s = cs[:, :1], cs[:, 1:]
        m, n = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
        y[..., m], y[..., n] = x[..., m] * c - x[..., n] * s, x[..., n] * c + x[..., m] * s
    return y


def plan(cached, added, free, free_count, table, page, capacity):
    """One token after another."""
    table = table.copy()
    stack = list(free[:max(0, min(free_count, len(free)))])
    slots, positions = np.full(capacity, -1, np.int64), np.zeros(capacity, np.int64)
    starts, lengths, status, n = [0], [], 0, 0
    short = 0
    for b, (c, a) in enumerate(zip(cached, added)):
        if c < 0 or a < 0:
            status |= 4
        c, a = max(c, 0), max(a, 0)
        if n + a > capacity:
            status |= 8
            a = capacity - n
        if c + a > table.shape[1] * page:
            status |= 2
        for i in range(a):
            pos = c + i
            positions[n] = pos
            if pos // page < table.shape[1]:
                if pos % page == 0:
                    if stack:
                        table[b, pos // page] = stack.pop()
                    else:
                        table[b, pos // page] = -1
                        status |= 1
                        short += 1
                if table[b, pos // page] >= 0:
                    slots[n] = table[b, pos // page] * page + pos % page
            n += 1
        starts.append(n)
        lengths.append(c + a)
    return dict(block_table=table, query_start=np.array(starts), kv_lengths=np.array(lengths), slots=slots,
                positions=positions, free_left=np.array([len(stack)]), status=np.array([status]))


def attention(q, k, v, scale, causal, window, cap, wide):
    """One request and kv head: q [rows, n, dim] (n query heads of a token), k and v [keys, dim] as stored (64 bits).
    Returns out, lse and a bound on each output's error before it is rounded.

    The bound. A score is a sum of dim products of f32 sums, each rounded by 2^-24 of the magnitudes M = scale |q| (|k|
    + range of k's codes), at most dim + 16 times, plus the exponential's argument (2^-24 of the score and of the
    reference) and result (2^-22): d relative error of each probability. Then out moves by at most 2 d max|v|. A
    probability times a value's scale is rounded to f16 (2^-11) beside magnitudes A = sum p (|v| + range); sums are f32
    over the keys. `wide` 1, as for prompts: the probability and the value are each rounded to f16 instead. `wide` 2, as
    for prompts in bf16 without lse: the key too, before the product (2^-11 of |k|, on scale |q| |k|), and the sum is of
    the rounded probabilities."""
    rows, n, dim = q.shape
    keys = k.shape[0]
    pos = keys - rows + np.arange(rows)[:, None]
    t = np.arange(keys)[None, :]
    seen = np.ones((rows, keys), bool)
    if causal:
        seen &= t <= pos
    if window:
        seen &= t > pos - window
    out, lse = np.zeros((rows, n, dim)), np.full((rows, n), -np.inf)
    tol = np.zeros((rows, n, dim))
    dlse = np.zeros((rows, n))
    if keys == 0:
        return out, lse, tol, dlse
    reach = 2 * np.abs(k).max(initial=0.0, where=np.isfinite(k))  # |s c| + |b| <= 3 max
    for h in range(n):
        with np.errstate(all="ignore"):
            x = q[:, h] @ k.T * scale
            mag = abs(scale) * (np.abs(q[:, h]) @ np.abs(k.T) + np.abs(q[:, h]).sum(-1, keepdims=True) * reach)
            wide_mag = abs(scale) * (np.abs(q[:, h]) @ np.abs(k.T)) * 2.0 ** -11 if wide == 2 else 0.0
            if cap:
                x = cap * np.tanh(x / cap)
        x = np.where(seen, x, -np.inf)
        any_seen = seen.any(-1)
        m = np.where(any_seen, x.max(-1), 0.0)
        with np.errstate(all="ignore"):
            p = np.where(seen, np.exp(x - m[:, None]), 0.0)
            total = p.sum(-1)
            vv = np.where(np.isfinite(v), v, 0.0)
            w = np.where(total[:, None] > 0, p / np.where(total > 0, total, 1.0)[:, None], 0.0)
            o = w @ vv
            # a value that is not a number reaches the rows that see it
            o = np.where((seen.astype(float) @ ~np.isfinite(v)) > 0, np.nan, o)
            o = np.where(np.isnan(np.where(seen, x, 0.0)).any(-1)[:, None], np.nan, o)
            d = np.where(seen, (dim + 16) * 2.0 ** -24 * mag + wide_mag + 2.0 ** -22 * (1 + np.abs(np.where(seen, x, 0.0)) +
                         np.abs(m[:, None])) + (2.0 ** -20 * cap if cap else 0.0), 0.0).max(-1)
            vmax = np.abs(vv).max(0)
            # |s c| of a value is at most |v| + |b|, and |b| at most the largest value of its group
            a = w @ (np.abs(vv) + np.abs(vv).max(-1, keepdims=True))
            tol[:, h] = 2 * d[:, None] * vmax[None] + a * (2.0 ** -11 + (2.0 ** -10 if wide else 0.0) +
                                                          (keys / 4 + 64) * 2.0 ** -24)
            lse[:, h] = np.where(any_seen, m + np.log(total), -np.inf)
            dlse[:, h] = d + (keys / 4 + 64) * 2.0 ** -24 + 2.0 ** -22 * (np.abs(m) + 4) + \
                (2.0 ** -11 if wide == 2 else 0.0)
        out[:, h] = o
    return out, lse, tol, dlse
