"""The 4-bit paged key/value cache as cases to be measured: the plan of a step
(block tables and slot maps from request lengths), the append of new key and
value rows with the rotary embedding before it, the read of rows back, and
attention over the cache.

`own` false: elementary torch operations on a cache in a plain layout (codes
two a byte, row by row, with f16 scale and bias planes). `own` true: the
calls of stark_amd.kv that a serving loop makes, arguments marshalled once.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LIMIT = 32768.0  # largest magnitude that a 4-bit group holds


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # A decode step of eight sequences, some of which need a new page: all launch and latency.
        dict(name="plan_decode_b8", family="plan", batch=8, page=64, ctx_lo=100, ctx_hi=4096, chunks=0, chunk=0),
        # A full server's step: 512 sequences, 24 of them with a prompt chunk of up to 500 tokens.
        dict(name="plan_mixed_b512", family="plan", batch=512, page=16, ctx_lo=1, ctx_hi=16384, chunks=24, chunk=500),
        # Decode of one sequence: one token's heads rotated, its key and value rows quantized.
        dict(name="append_decode_t1", family="append", tokens=1, heads=32, kv_heads=8, dim=128, group=64, page=64,
             dtype="bf16", axes=1, rotary=128),
        # A prompt chunk with image positions on three axes (time, height, width).
        dict(name="append_axes3_t2048", family="append", tokens=2048, heads=32, kv_heads=8, dim=128, group=64,
             page=64, dtype="bf16", axes=3, rotary=128),
        # f32 rows (the hybrid engine's activations), an odd count, half of each head rotated, small groups.
        dict(name="append_f32_t1531", family="append", tokens=1531, heads=12, kv_heads=4, dim=64, group=32, page=16,
             dtype="f32", axes=1, rotary=32),
        # A cached prefix of 8192 tokens taken out in bf16, as for a model that shares it without 4-bit attention.
        dict(name="read_t8192", family="read", tokens=8192, kv_heads=8, dim=128, group=64, page=64, dtype="bf16"),
        # A few hundred rows of wide heads in f16.
        dict(name="read_dim256_t333", family="read", tokens=333, kv_heads=2, dim=256, group=128, page=32,
             dtype="f16"),
        # Decode of one sequence at the end-to-end benchmark's context.
        dict(name="attend_decode_b1_ctx4096", family="attend", batch=1, q_lo=1, q_hi=1, ctx_lo=4096, ctx_hi=4096,
             heads=32, kv_heads=8, dim=128, group=64, page=64, dtype="bf16", window=0, cap=0.0, lse=False),
        # Decode of a full batch of unlike lengths.
        dict(name="attend_decode_b64", family="attend", batch=64, q_lo=1, q_hi=1, ctx_lo=500, ctx_hi=32768, heads=32,
             kv_heads=8, dim=128, group=64, page=64, dtype="bf16", window=0, cap=0.0, lse=False),
        # Speculative verify: drafts of up to five tokens, eight query heads to a key head, small pages.
        dict(name="attend_verify_b16", family="attend", batch=16, q_lo=2, q_hi=5, ctx_lo=900, ctx_hi=9000, heads=32,
             kv_heads=4, dim=128, group=32, page=16, dtype="bf16", window=0, cap=0.0, lse=True),
        # A prefill chunk of 2048 tokens behind 4096 cached ones: the largest call.
        dict(name="attend_chunk_t2048", family="attend", batch=1, q_lo=2048, q_hi=2048, ctx_lo=4096, ctx_hi=4096,
             heads=32, kv_heads=8, dim=128, group=64, page=64, dtype="bf16", window=0, cap=0.0, lse=False),
        # Prompts and decode rows of a hybrid layer together: f16, heads of 64, a sliding window, soft-capped scores.
        dict(name="attend_mixed_f16", family="attend", batch=12, q_lo=1, q_hi=701, ctx_lo=1, ctx_hi=3001, heads=16,
             kv_heads=8, dim=64, group=32, page=32, dtype="f16", window=1024, cap=30.0, lse=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8])
    return kv * rng.choice([1, 2, 4, 5, 7, 8]), kv


def draw(rng):
    family = rng.choice(["plan", "append", "append", "read", "attend", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128])
    dim = rng.choice([64, 128, 128, 256])
    group = rng.choice([g for g in (32, 64, 128) if g <= dim])
    if family == "plan":
        batch = _log(rng, 1, 1024)
        return dict(family=family, batch=batch, page=page, ctx_lo=1, ctx_hi=_log(rng, 16, 16384),
                    chunks=rng.randint(0, min(batch, 16)), chunk=_log(rng, 2, 1000))
    heads, kv = _heads(rng)
    if family == "append":
        axes = rng.choice([0, 1, 1, 3])
        return dict(family=family, tokens=_log(rng, 1, 4096), heads=heads, kv_heads=kv, dim=dim, group=group,
                    page=page, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), axes=axes,
                    rotary=dim if axes != 1 else rng.choice([dim, dim // 2]))
    if family == "read":
        return dict(family=family, tokens=_log(rng, 1, 8192), kv_heads=kv, dim=dim, group=group, page=page,
                    dtype=rng.choice(["bf16", "f16", "f32"]))
    kind = rng.choice(["decode", "decode", "verify", "prompt", "mixed"])
    if kind == "decode":
        batch, q_lo, q_hi, hi = _log(rng, 1, 64), 1, 1, _log(rng, 16, 16384)
    elif kind == "verify":
        batch, q_lo, q_hi, hi = _log(rng, 1, 32), 1, rng.randint(2, 8), _log(rng, 16, 8192)
    elif kind == "prompt":
        batch, q_lo, hi = rng.randint(1, 3), 1, _log(rng, 1, 2048)
        q_hi = _log(rng, 17, 1000)
    else:
        batch, q_lo, hi = rng.randint(2, 12), 1, _log(rng, 1, 2048)
        q_hi = _log(rng, 2, 250)
    return dict(family="attend", batch=batch, q_lo=q_lo, q_hi=q_hi, ctx_lo=1, ctx_hi=hi, heads=min(heads, 32),
                kv_heads=kv, dim=dim, group=group, page=page, dtype=rng.choice(["bf16", "bf16", "f16"]),
                window=rng.choice([0, 0, 0, _log(rng, 16, 2048)]), cap=rng.choice([0.0, 0.0, 30.0]),
                lse=rng.choice([False, True]))


def _lengths(case):
    """Cached and new tokens of each request: fixed by the case."""
    r = random.Random("%d %d %d" % (case["batch"], case["ctx_lo"], case["ctx_hi"]))
    if case["family"] == "plan":
        cached = [_log(r, case["ctx_lo"], case["ctx_hi"]) for _ in range(case["batch"])]
        added = [1] * case["batch"]
        for b in r.sample(range(case["batch"]), case["chunks"]):
            added[b] = r.randint(1, case["chunk"])
        return cached, added
    cached = [_log(r, case["ctx_lo"], case["ctx_hi"]) for _ in range(case["batch"])]
    added = [_log(r, case["q_lo"], case["q_hi"]) for _ in range(case["batch"])]
    return cached, added


def _axis_of_pair(case):
    """The position axis of each rotated pair: sections in the ratio 2 : 3 : 3 for three axes."""
    pairs = case["rotary"] // 2
    if case["axes"] <= 1:
        return [0] * pairs
    a, b = pairs // 4, pairs // 4 + 3 * pairs // 8
    return [0 if i < a else 1 if i < b else 2 for i in range(pairs)]


# ---------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _keys(gen, tokens, kv_heads, dim):
    """Key rows: a few channels of each head carry an offset and a wider spread, as rotated keys have."""
    spread = torch.exp(0.5 * _randn(gen, 1, kv_heads, dim))
    offset = _randn(gen, 1, kv_heads, dim) * (torch.rand(1, kv_heads, dim, generator=gen, device="cuda") < 0.1) * 4.0
    return _randn(gen, tokens, kv_heads, dim) * spread + offset


def _quantize(x, group):
    """Codes [.., dim] u8, scales and biases [.., dim / group] f16 of rows; in 64 bits, for 32 take values half
    way between two codes to the wrong one."""
    g = x.double().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1), g.amax(-1)
    bad = ~((lo >= -LIMIT) & (hi <= LIMIT))
    s = ((hi - lo) / 15.0).half()
    b = lo.half()
    sf, bf = s.double().unsqueeze(-1), b.double().unsqueeze(-1)
    q = torch.round((g - bf) / torch.where(sf > 0, sf, torch.ones_like(sf)))
    q = torch.where((sf > 0) & ~bad.unsqueeze(-1), q, torch.zeros_like(q)).clamp_(0, 15).to(torch.uint8)
    nan = torch.full_like(s, float("nan"))
    return q.flatten(-2), torch.where(bad, nan, s), torch.where(bad, nan, b)


def _pack(q):
    return q[..., 0::2] | (q[..., 1::2] << 4)


def _values(codes, s, b):
    """f32 rows of packed codes and planes."""
    q = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    q = q.unflatten(-1, (s.shape[-1], -1)).float()
    return (q * s.float().unsqueeze(-1) + b.float().unsqueeze(-1)).flatten(-2)


class _PlainCache:
    """codes [slots, 2, kv_heads, dim / 2] u8; planes [slots, 2, kv_heads, groups] f16 (second axis: key, value)."""

    def __init__(self, slots, kv_heads, dim, group):
        self.group = group
        self.codes = torch.zeros(slots, 2, kv_heads, dim // 2, dtype=torch.uint8, device="cuda")
        self.s = torch.zeros(slots, 2, kv_heads, dim // group, dtype=torch.float16, device="cuda")
        self.b = torch.zeros_like(self.s)

    def append(self, slots, k, v):
        for i, x in enumerate((k, v)):
            q, s, b = _quantize(x, self.group)
            self.codes[slots, i], self.s[slots, i], self.b[slots, i] = _pack(q), s, b

    def rows(self, slots, i):
        return _values(self.codes[slots, i], self.s[slots, i], self.b[slots, i])


def _fill(gen, cache, slots, kv_heads, dim, dtype):
    """Key and value rows of the type, written at the slots in pieces."""
    for at in slots.split(65536):
        k, v = _keys(gen, at.numel(), kv_heads, dim).to(dtype), _randn(gen, at.numel(), kv_heads, dim).to(dtype)
        if own:
            from stark_amd import kv as KV
            KV.KvAppend(cache, k=k, v=v, slots=at.int()).encode()
            torch.cuda.current_stream().synchronize()
        else:
            cache.append(at, k, v)


def _make_cache(case, pages):
    if own:
        from stark_amd import kv as KV
        return KV.KvCache(pages, case["page"], case["kv_heads"], case["dim"], case["group"])
    return _PlainCache(pages * case["page"], case["kv_heads"], case["dim"], case["group"])


def _pages(case, cached, added):
    return [-(-(c + a) // case["page"]) for c, a in zip(cached, added)]


def prepare(case, seed):
    gen = _gen(seed)
    if case["family"] == "plan":
        return _prepare_plan(case, gen)
    if case["family"] == "append":
        return _prepare_append(case, gen)
    if case["family"] == "read":
        return _prepare_read(case, gen)
    return _prepare_attend(case, gen)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _prepare_plan(case, gen):
    cached, added = _lengths(case)
    page, total = case["page"], sum(added)
    have, need = [-(-c // page) for c in cached], _pages(case, cached, added)
    pages = sum(need) + 64
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    table = torch.full((case["batch"], max(need) + 8), -1, dtype=torch.int32, device="cuda")
    row = torch.repeat_interleave(torch.arange(case["batch"], device="cuda"), torch.tensor(have, device="cuda"))
    start = torch.tensor([sum(have[:b]) for b in range(case["batch"])], device="cuda")
    table[row, torch.arange(sum(have), device="cuda") - start[row]] = order[:sum(have)]
    state = dict(family="plan", page=page, cached=_ints(cached), added=_ints(added), table=table, total=total,
                 free=order[sum(have):].contiguous(), free_count=_ints([pages - sum(have)]), capacity=total + 8)
    if own:
        from stark_amd import kv as KV
        state["op"] = KV.KvPlan(state["cached"], state["added"], state["free"], state["free_count"], table, page,
                                state["capacity"])
    return state


def _prepare_append(case, gen):
    t, h, kv, dim, dtype = case["tokens"], case["heads"], case["kv_heads"], case["dim"], DT[case["dtype"]]
    pages = -(-t // case["page"]) + 3
    # the new rows follow a short prefix in pages of any order
    order = torch.randperm(pages, generator=gen, device="cuda")
    at = torch.arange(t, device="cuda") + 5 % case["page"]
    slots = order[at // case["page"]] * case["page"] + at % case["page"]
    state = dict(family="append", q=_randn(gen, t, h, dim).to(dtype), k=_keys(gen, t, kv, dim).to(dtype),
                 v=_randn(gen, t, kv, dim).to(dtype), slots=slots, case=case, cache=_make_cache(case, pages))
    if case["axes"]:
        pairs, rows = case["rotary"] // 2, 8192
        freq = 1e6 ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
        angle = torch.arange(rows, dtype=torch.float64, device="cuda").unsqueeze(1) * freq
        state["table"] = torch.stack([angle.cos(), angle.sin()], dim=-1).float().contiguous()
        first = torch.randint(0, rows - t, (1,), generator=gen, device="cuda")
        p = torch.arange(t, device="cuda") + first
        # three axes: frames of 24 by 32 patches
        state["positions"] = torch.stack([p] if case["axes"] == 1 else
                                         [p // 768, p // 32 % 24, p % 32]).int().contiguous()
        state["axis"] = _axis_of_pair(case)
        state["axis_index"] = torch.tensor(state["axis"], device="cuda")
    if own:
        from stark_amd import kv as KV
        state["q_out"] = torch.empty_like(state["q"])
        rot = KV.Rotary(state["table"], state["positions"], state["axis"]) if case["axes"] else None
        at = slots.int()
        state["op"] = KV.KvAppend(state["cache"], k=state["k"], v=state["v"], slots=at, q=state["q"],
                                  q_out=state["q_out"], rotary=rot)
        state["k_out"] = torch.empty(t, kv, dim, device="cuda")
        state["v_out"] = torch.empty_like(state["k_out"])
        state["read"] = KV.KvRead(state["cache"], at, state["k_out"], state["v_out"])
    return state


def _prepare_read(case, gen):
    t = case["tokens"]
    pages = -(-t // case["page"])
    order = torch.randperm(pages, generator=gen, device="cuda")
    at = torch.arange(t, device="cuda")
    slots = order[at // case["page"]] * case["page"] + at % case["page"]
    cache = _make_cache(case, pages)
    _fill(gen, cache, slots, case["kv_heads"], case["dim"], torch.bfloat16)
    state = dict(family="read", cache=cache, slots=slots, dtype=DT[case["dtype"]])
    if own:
        from stark_amd import kv as KV
        state["k_out"] = torch.empty(t, case["kv_heads"], case["dim"], dtype=state["dtype"], device="cuda")
        state["v_out"] = torch.empty_like(state["k_out"])
        state["op"] = KV.KvRead(cache, slots.int(), state["k_out"], state["v_out"])
    return state


def _prepare_attend(case, gen):
    cached, added = _lengths(case)
    need, page, dim, dtype = _pages(case, cached, added), case["page"], case["dim"], DT[case["dtype"]]
    order = torch.randperm(sum(need), generator=gen, device="cuda").int()
    table = torch.full((case["batch"], max(need)), -1, dtype=torch.int32, device="cuda")
    slots, start = [], 0
    for b, n in enumerate(need):
        ids = order[start:start + n]
        table[b, :n] = ids
        at = torch.arange(cached[b] + added[b], device="cuda")
        slots.append(ids.long()[at // page] * page + at % page)
        start += n
    cache = _make_cache(case, sum(need))
    _fill(gen, cache, torch.cat(slots), case["kv_heads"], dim, dtype)
    q = (_randn(gen, sum(added), case["heads"], dim) * 1.5).to(dtype)
    qs = [0]
    for a in added:
        qs.append(qs[-1] + a)
    state = dict(family="attend", case=case, cache=cache, q=q, slots=slots, cached=cached, added=added,
                 table=table, query_start=_ints(qs), kv_lengths=_ints([c + a for c, a in zip(cached, added)]))
    if own:
        from stark_amd import kv as KV
        state["out"] = torch.empty_like(q)
        state["lse"] = torch.empty(q.shape[:2], device="cuda") if case["lse"] else None
        state["op"] = KV.KvAttention(cache, q, state["out"], table, state["query_start"], state["kv_lengths"],
                                     max_query=max(added), max_kv=max(c + a for c, a in zip(cached, added)),
                                     window=case["window"], soft_cap=case["cap"], lse=state["lse"])
    return state


# ---------------------------------------------------------------- one pass

def run(state):
    if own:
        return _run_own(state)
    return {"plan": _run_plan, "append": _run_append, "read": _run_read, "attend": _run_attend}[state["family"]](state)


def _run_own(state):
    op = state["op"]
    op.encode()
    if state["family"] == "plan":
        return dict(block_table=state["table"], query_start=op.query_start, kv_lengths=op.kv_lengths, slots=op.slots,
                    positions=op.positions, free_left=op.free_left, status=op.status)
    if state["family"] == "append":
        state["read"].encode()
        return dict(q=state["q_out"], k=state["k_out"], v=state["v_out"])
    if state["family"] == "read":
        return dict(k=state["k_out"], v=state["v_out"])
    return dict(out=state["out"]) if state["lse"] is None else dict(out=state["out"], lse=state["lse"])


def _run_plan(s):
    cached, added, page, table = s["cached"].long(), s["added"].long(), s["page"], s["table"]
    batch = cached.numel()
    zero = torch.zeros(1, dtype=torch.int64, device="cuda")
    query_start = torch.cat([zero, added.cumsum(0)])
    lengths = cached + added
    before, after = (cached + page - 1) // page, (lengths + page - 1) // page
    page_start = torch.cat([zero, (after - before).cumsum(0)])
    # new page j comes off the end of the free list
    j = torch.arange(s["free"].numel(), device="cuda")
    owner = torch.searchsorted(page_start, j, right=True) - 1
    used = owner < batch
    owner = owner.clamp(max=batch - 1)
    ids = s["free"].long()[(s["free_count"].long() - 1 - j).clamp(min=0)]
    ids = torch.where(j < s["free_count"], ids, -1)
    column = before[owner] + j - page_start[owner]
    flat = table.view(-1)
    where = torch.where(used, owner * table.shape[1] + column, 0)
    flat.index_put_((where,), torch.where(used, ids, flat[where].long()).int())
    n = torch.arange(s["capacity"], device="cuda")
    req = torch.searchsorted(query_start, n, right=True) - 1
    live = req < batch
    req = req.clamp(max=batch - 1)
    pos = cached[req] + n - query_start[req]
    pid = table.long()[req, torch.where(live, pos // page, 0)]
    slots = torch.where(live & (pid >= 0), pid * page + pos % page, -1)
    taken = page_start[-1:]
    left = (s["free_count"].long() - taken).clamp(min=0)
    return dict(block_table=table, query_start=query_start.int(), kv_lengths=lengths.int(), slots=slots.int(),
                positions=torch.where(live, pos, 0).int(), free_left=left.int(),
                status=(taken > s["free_count"]).int())


def _rotate(x, s):
    """64-bit rows with their first `rotary` values rotated in pairs (i, i + rotary / 2)."""
    pairs = s["axis_index"].numel()
    cs = s["table"].double()[s["positions"].long()[s["axis_index"]].t(), torch.arange(pairs, device="cuda")]
    c, n = cs[..., 0].unsqueeze(1), cs[..., 1].unsqueeze(1)
    a, b = x[..., :pairs], x[..., pairs:2 * pairs]
    return torch.cat([a * c - b * n, b * c + a * n, x[..., 2 * pairs:]], dim=-1)


def _run_append(s):
    q, k = s["q"].double(), s["k"].double()
    if s["case"]["axes"]:
        q, k = _rotate(q, s), _rotate(k, s)
    s["cache"].append(s["slots"], k, s["v"])
    return dict(q=q.to(s["q"].dtype), k=s["cache"].rows(s["slots"], 0), v=s["cache"].rows(s["slots"], 1))


def _run_read(s):
    return dict(k=s["cache"].rows(s["slots"], 0).to(s["dtype"]), v=s["cache"].rows(s["slots"], 1).to(s["dtype"]))


def _run_attend(s):
    case = s["case"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    out = torch.empty_like(s["q"])
    lse = torch.empty(s["q"].shape[:2], device="cuda")
    start = 0
    for b, (c, a) in enumerate(zip(s["cached"], s["added"])):
        k, v = (s["cache"].rows(s["slots"][b], i).transpose(0, 1) for i in (0, 1))  # [kv, tokens, dim]
        q = s["q"][start:start + a].float().view(a, kv, heads // kv, dim).permute(1, 2, 0, 3).reshape(kv, -1, dim)
        x = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(dim)
        if case["cap"]:
            x = case["cap"] * torch.tanh(x / case["cap"])
        pos = (c + torch.arange(a, device="cuda")).repeat(heads // kv).unsqueeze(1)
        t = torch.arange(c + a, device="cuda")
        seen = t <= pos
        if case["window"]:
            seen &= t > pos - case["window"]
        x = x.masked_fill(~seen, float("-inf"))
        m = x.amax(-1, keepdim=True)
        p = torch.exp(x - m)
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p, v.contiguous()) / total
        out[start:start + a] = o.view(kv, heads // kv, a, dim).permute(2, 0, 1, 3).reshape(a, heads, dim).to(out.dtype)
        lse[start:start + a] = (m + total.log()).view(heads, a).t()
        start += a
    return dict(out=out, lse=lse) if case["lse"] else dict(out=out)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    size = 4 if case.get("dtype") == "f32" else 2
    if case["family"] == "plan":
        cached, added = _lengths(case)
        new = sum(_pages(case, cached, added)) - sum(-(-c // case["page"]) for c in cached)
        return {"bytes": 4 * (case["batch"] * 5 + 2 * new + 2 * sum(added)), "flops": 0}
    row = case["kv_heads"] * (case["dim"] // 2 + 4 * (case["dim"] // case["group"]))  # bytes of one key (or value) row
    if case["family"] == "append":
        t, d = case["tokens"], case["dim"]
        moved = t * d * size * (2 * case["heads"] + 2 * case["kv_heads"]) + t * (4 + 4 * case["axes"])
        return {"bytes": moved + t * (2 * row * 2 + 2 * 4 * case["kv_heads"] * d) +
                (8 * t * case["rotary"] // 2 if case["axes"] else 0), "flops": 0}
    if case["family"] == "read":
        return {"bytes": case["tokens"] * (2 * row + 2 * size * case["kv_heads"] * case["dim"] + 4), "flops": 0}
    cached, added = _lengths(case)
    seen = tokens = 0
    for c, a in zip(cached, added):
        w = case["window"] or c + a
        seen += sum(min(c + i + 1, w) for i in range(a))
        tokens += min(c + a, w + a - 1)
    io = 2 * size * sum(added) * case["heads"] * case["dim"] + (4 * sum(added) * case["heads"] if case["lse"] else 0)
    return {"bytes": 2 * row * tokens + io, "flops": 4 * seen * case["heads"] * case["dim"]}


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_rows(x, group):
    """What 4 bits a value hold of 64-bit rows: f16 planes, codes to the nearest step."""
    out = torch.empty_like(x)
    for at in range(0, x.shape[-1], group):
        g = x[..., at:at + group]
        low, high = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
        step, base = ((high - low) / 15).half().double(), low.half().double()
        code = torch.where(step > 0, ((g - base) / step).round().clamp(0, 15), 0.0)
        out[..., at:at + group] = base + step * code
    return out


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    if case["family"] == "plan":
        return None
    if case["family"] == "append":
        q, k, v = (s[n].double() for n in ("q", "k", "v"))
        if case["axes"]:
            pairs = case["rotary"] // 2
            for i, axis in enumerate(s["axis"]):
                cs = s["table"].double()[s["positions"][axis].long(), i]
                turn = torch.complex(cs[:, 0], cs[:, 1]).unsqueeze(1)
                for x in (q, k):
                    z = torch.complex(x[..., i].clone(), x[..., i + pairs].clone()) * turn
                    x[..., i], x[..., i + pairs] = z.real, z.imag
        return dict(q=q, k=_exact_rows(k, case["group"]), v=_exact_rows(v, case["group"]))
    cache = s["cache"]

    def stored(slots, i):
        codes = cache.codes[slots, i].to(torch.int64)
        full = torch.empty(*codes.shape[:-1], case["dim"], dtype=torch.float64, device="cuda")
        full[..., 0::2], full[..., 1::2] = (codes % 16).double(), (codes // 16).double()
        step = cache.s[slots, i].double().repeat_interleave(case["group"], -1)
        return full * step + cache.b[slots, i].double().repeat_interleave(case["group"], -1)

    if case["family"] == "read":
        return dict(k=stored(s["slots"], 0), v=stored(s["slots"], 1))
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    each = case["heads"] // case["kv_heads"]
    first = 0
    for b, (c, a) in enumerate(zip(s["cached"], s["added"])):
        keys, vals = stored(s["slots"][b], 0), stored(s["slots"][b], 1)
        behind = (c + torch.arange(a, device="cuda"))[:, None] - torch.arange(c + a, device="cuda")[None, :]
        hidden = behind < 0
        if case["window"]:
            hidden = hidden | (behind >= case["window"])
        for h in range(case["heads"]):
            x = (s["q"][first:first + a, h].double() @ keys[:, h // each].t()) * case["dim"] ** -0.5
            if case["cap"]:
                x = torch.tanh(x / case["cap"]) * case["cap"]
            x[hidden] = float("-inf")
            total = torch.logsumexp(x, -1)
            out[first:first + a, h] = torch.exp(x - total[:, None]) @ vals[:, h // each]
            lse[first:first + a, h] = total
        first += a
    return dict(out=out, lse=lse) if case["lse"] else dict(out=out)
