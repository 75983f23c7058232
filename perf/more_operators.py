"""Products of 8-bit floating-point weights as cases to be measured: the plan of a
step's routed experts, rows to e4m3 with a scale for each 128 values, the product
with weights that have a scale for each 128 x 128 block, the same grouped by expert,
and the weighted sum of a token's expert rows.

`own` false: elementary torch operations. `own` true: the calls of stark_amd.fp8 that
a serving loop makes, arguments marshalled once.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
F8 = torch.float8_e4m3fn
BLOCK = 128
LARGEST = 448.0  # of e4m3
SMALLEST_SCALE = 2.0 ** -126


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # Routes of a decode step of 16 sequences, eight of 128 experts each: launch and latency.
        dict(name="plan_decode_t16", family="plan", tokens=16, active=8, experts=128, first=0, routed=128),
        # Routes of a prompt of 8192 tokens.
        dict(name="plan_prompt_t8192", family="plan", tokens=8192, active=8, experts=128, first=0, routed=128),
        # Activations of a decode step before a layer's products.
        dict(name="quantize_decode_t16", family="quantize", rows=16, columns=4096, dtype="bf16", gated=False, blocks_first=False),
        # The gated activations of a prompt's routed rows, between the experts' two products.
        dict(name="quantize_gated_r65536", family="quantize", rows=65536, columns=768, dtype="bf16", gated=True, blocks_first=False),
        # Decode of one sequence: the up projection of a dense layer.
        dict(name="matmul_decode_m1", family="matmul", m=1, n=12288, k=4096, dtype="bf16", bias=False, blocks_first=False),
        # Speculative verify: five rows through the down projection, f16 with a bias.
        dict(name="matmul_verify_m5", family="matmul", m=5, n=4096, k=12288, dtype="f16", bias=True, blocks_first=False),
        # Odd sizes: a ragged batch, a matrix that ends inside a tile and inside a block, f32 out.
        dict(name="matmul_ragged_m333", family="matmul", m=333, n=1001, k=2000, dtype="f32", bias=True, blocks_first=False),
        # A prompt of 4096 tokens through the up projection.
        dict(name="matmul_prompt_m4096", family="matmul", m=4096, n=12288, k=4096, dtype="bf16", bias=False, blocks_first=False),
        # 16 sequences, eight of 128 experts each: one or two rows to an expert.
        dict(name="grouped_decode_t16", family="grouped", tokens=16, active=8, experts=128, n=1536, k=2048, dtype="bf16", gather=True,
             spare=0, blocks_first=False),
        # A prompt of 8192 tokens, 512 rows to an expert on average: the largest call.
        dict(name="grouped_prompt_t8192", family="grouped", tokens=8192, active=8, experts=128, n=1536, k=2048, dtype="bf16", gather=True,
             spare=0, blocks_first=False),
        # Decode: the rows of 16 sequences' experts back to their tokens.
        dict(name="combine_decode_t16", family="combine", tokens=16, active=8, width=2048, dtype="bf16", kept=1.0),
        # The same of a prompt.
        dict(name="combine_prompt_t8192", family="combine", tokens=8192, active=8, width=2048, dtype="bf16", kept=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _columns(rng, lo, hi):
    """Whole blocks, whole 16-byte pieces, or any."""
    k = _log(rng, lo, hi)
    unit = rng.choice([128, 128, 16, 1])
    return max(1, k // unit) * unit


def draw(rng):
    family = rng.choice(["plan", "quantize", "matmul", "matmul", "matmul", "grouped", "grouped", "combine"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    blocks_first = rng.choice([False, False, True])
    if family == "plan":
        routed = _log(rng, 1, 512)
        experts = rng.choice([routed, max(1, routed // 4)])  # all of them, or one rank's share
        return dict(family=family, tokens=_log(rng, 1, 8192), active=rng.randint(1, min(8, routed)), experts=experts,
                    first=rng.choice([0, routed - experts]), routed=routed)
    if family == "quantize":
        return dict(family=family, rows=_log(rng, 1, 16384), columns=_columns(rng, 32, 4096), dtype=dtype,
                    gated=rng.choice([False, True]), blocks_first=blocks_first)
    if family == "matmul":
        kind = rng.choice(["decode", "verify", "prompt"])
        m = {"decode": 1, "verify": rng.randint(2, 16), "prompt": _log(rng, 17, 4096)}[kind]
        return dict(family=family, m=m, n=_log(rng, 16, 8192), k=_columns(rng, 64, 8192), dtype=dtype, bias=rng.choice([False, True]),
                    blocks_first=blocks_first)
    if family == "grouped":
        experts = _log(rng, 1, 128)
        return dict(family=family, tokens=_log(rng, 1, 2048), active=rng.randint(1, min(8, experts)), experts=experts,
                    n=_log(rng, 64, 2048), k=_columns(rng, 64, 2048), dtype=dtype, gather=rng.choice([False, True]),
                    spare=rng.choice([0, 0, 37]), blocks_first=blocks_first)
    return dict(family=family, tokens=_log(rng, 1, 4096), active=rng.randint(1, 8), width=_log(rng, 64, 4096), dtype=dtype,
                kept=rng.choice([1.0, 1.0, 0.3]))


def _group_sizes(case):
    """Rows of each expert, fixed by the case: experts are not equally liked, and a token takes one once."""
    r = np.random.RandomState((case["tokens"] * 31 + case["experts"]) % (1 << 31))
    liked = 0.6 * r.randn(case["experts"])
    score = liked + r.gumbel(size=(case["tokens"], case["experts"]))
    ids = np.argsort(-score, axis=1)[:, :case["active"]]
    return np.bincount(ids.ravel(), minlength=case["experts"]).tolist()


# ---------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _blocks(n):
    return -(-n // BLOCK)


def _codes(gen, *shape):
    """e4m3 codes of normally distributed values, each row at a whole number of 16-byte pieces from the last."""
    wide = -(-shape[-1] // 16) * 16
    x = (_randn(gen, *shape[:-1], wide) * 110.0).clamp_(-LARGEST, LARGEST).to(F8)
    return x[..., :shape[-1]]


def _row_scales(gen, rows, k, blocks_first):
    """A scale for each row and block; a few rows are far larger, as activations are."""
    s = 0.01 * torch.exp(0.4 * _randn(gen, rows, _blocks(k)) + 2.0 * (_randn(gen, rows, 1) > 2.0))
    return s.t().contiguous().t() if blocks_first else s


def _weights(gen, lead, n, k):
    scales = 2e-4 * torch.exp(0.3 * _randn(gen, *lead, _blocks(n), _blocks(k)))
    return _codes(gen, *lead, n, k), scales


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = _gen(seed)
    state = {"plan": _prepare_plan, "quantize": _prepare_quantize, "matmul": _prepare_matmul, "grouped": _prepare_grouped,
             "combine": _prepare_combine}[case["family"]](case, gen)
    state["case"] = case
    if own:
        state["op"] = _operator(state)
    return state


def _operator(s):
    """The framework's operator on the state's tensors."""
    from stark_amd import fp8
    case = s["case"]
    if case["family"] == "plan":
        return fp8.ExpertPlan(s["ids"], case["experts"], case["first"])
    if case["family"] == "quantize":
        return fp8.Fp8Quantize(s["x"], s["codes"], s["scales"], gated=case["gated"])
    if case["family"] == "matmul":
        return fp8.Fp8Matmul(s["a"], s["a_scales"], s["b"], s["b_scales"], s["d"], bias=s["bias"])
    if case["family"] == "grouped":
        return fp8.Fp8GroupedMatmul(s["a"], s["a_scales"], s["b"], s["b_scales"], s["d"], s["group_start"], a_rows=s["a_rows"])
    return fp8.ExpertCombine(s["x"], s["slots"], s["weights"], s["out"])


def _prepare_plan(case, gen):
    liked = 0.6 * _randn(gen, 1, case["routed"])
    u = torch.rand(case["tokens"], case["routed"], generator=gen, device="cuda").clamp_(1e-12, 1.0)
    ids = (liked - (-u.log()).clamp_(min=1e-12).log()).topk(case["active"], dim=1).indices
    return dict(ids=ids.int().contiguous())


def _prepare_quantize(case, gen):
    rows, k, dtype = case["rows"], case["columns"], DT[case["dtype"]]
    # rows of unlike size, a few channels far above the rest
    x = _randn(gen, rows, k * (2 if case["gated"] else 1)) * torch.exp(0.5 * _randn(gen, rows, 1))
    x *= 1.0 + 20.0 * (torch.rand(1, x.shape[1], generator=gen, device="cuda") < 0.005)
    scales = torch.empty(_blocks(k), rows, device="cuda").t() if case["blocks_first"] else torch.empty(rows, _blocks(k), device="cuda")
    return dict(x=x.to(dtype), codes=torch.zeros(rows, -(-k // 16) * 16, dtype=torch.uint8, device="cuda").view(F8)[:, :k], scales=scales)


def _prepare_matmul(case, gen):
    m, n, k, dtype = case["m"], case["n"], case["k"], DT[case["dtype"]]
    b, b_scales = _weights(gen, (), n, k)
    return dict(a=_codes(gen, m, k), a_scales=_row_scales(gen, m, k, case["blocks_first"]), b=b, b_scales=b_scales,
                bias=_randn(gen, n).to(dtype) if case["bias"] else None, d=torch.zeros(m, n, dtype=dtype, device="cuda"))


def _prepare_grouped(case, gen):
    sizes, n, k, tokens = _group_sizes(case), case["n"], case["k"], case["tokens"]
    total = sum(sizes)
    start = [0]
    for s in sizes:
        start.append(start[-1] + s)
    expert = torch.repeat_interleave(torch.arange(case["experts"], device="cuda"), torch.tensor(sizes, device="cuda"))
    token = (expert * tokens + torch.randint(0, tokens, (total,), generator=gen, device="cuda")).sort().values % tokens
    a_rows = torch.cat([token.int(), _ints([-1] * case["spare"])]) if case["gather"] else None
    count = tokens if case["gather"] else total + case["spare"]
    b, b_scales = _weights(gen, (case["experts"],), n, k)
    return dict(a=_codes(gen, count, k), a_scales=_row_scales(gen, count, k, case["blocks_first"]), b=b, b_scales=b_scales, a_rows=a_rows,
                group_start=_ints(start), d=torch.zeros(total + case["spare"], n, dtype=DT[case["dtype"]], device="cuda"), total=total,
                most=max(sizes))


def _prepare_combine(case, gen):
    tokens, active, dtype = case["tokens"], case["active"], DT[case["dtype"]]
    routes = tokens * active
    kept = torch.rand(routes, generator=gen, device="cuda") < case["kept"]  # the other routes are another rank's
    place = torch.randperm(routes, generator=gen, device="cuda")
    weights = torch.softmax(_randn(gen, tokens, active), dim=1)
    return dict(x=_randn(gen, routes, case["width"]).to(dtype), slots=torch.where(kept, place, -1).int().view(tokens, active),
                weights=weights, out=torch.zeros(tokens, case["width"], dtype=dtype, device="cuda"))


# ---------------------------------------------------------------- one pass

def run(state):
    if own:
        return _run_own(state)
    return {"plan": _run_plan, "quantize": _run_quantize, "matmul": _run_matmul, "grouped": _run_grouped,
            "combine": _run_combine}[state["case"]["family"]](state)


def _run_own(s):
    op, family = s["op"], s["case"]["family"]
    op.encode()
    if family == "plan":
        return dict(group_start=op.group_start, tokens=op.tokens, slots=op.slots)
    if family == "quantize":
        return dict(codes=s["codes"], scales=s["scales"])
    return dict(out=s["out"]) if family == "combine" else dict(d=s["d"])


def _run_plan(s):
    case, ids = s["case"], s["ids"].long().view(-1)
    experts = case["experts"]
    e = ids - case["first"]
    e = torch.where((e >= 0) & (e < experts), e, experts)
    got = torch.sort(e, stable=True)
    group_start = torch.searchsorted(got.values, torch.arange(experts + 1, device="cuda"))
    here = got.values < experts
    tokens = torch.where(here, got.indices // case["active"], -1)
    slots = torch.empty_like(e)
    slots[got.indices] = torch.where(here, torch.arange(e.numel(), device="cuda"), -1)
    return dict(group_start=group_start.int(), tokens=tokens.int(), slots=slots.int().view(s["ids"].shape))


def _activations(s):
    """64-bit values that are to be held in 8 bits."""
    x = s["x"].double()
    if not s["case"]["gated"]:
        return x
    k = s["case"]["columns"]
    return x[:, :k] * (x[:, k:] / (1.0 + torch.exp(-x[:, k:])))


def _run_quantize(s):
    x = _activations(s)
    rows, k = x.shape
    x = torch.nn.functional.pad(x, (0, _blocks(k) * BLOCK - k)).view(rows, -1, BLOCK)
    scale = (x.abs().amax(-1) / LARGEST).float().clamp_(min=SMALLEST_SCALE)
    q = x / scale.double().unsqueeze(-1)
    # the step of a value's binade: three bits behind its first, from 2^-9 on
    binade = ((q.abs().view(torch.int64) >> 52) << 52).view(torch.float64).clamp_(min=2.0 ** -6)
    q = (torch.round(q / (binade / 8)) * (binade / 8)).clamp_(-LARGEST, LARGEST)
    s["codes"].copy_(q.view(rows, -1)[:, :k].float())
    s["scales"].copy_(scale)
    return dict(codes=s["codes"], scales=s["scales"])


def _spread(scales, n):
    """A scale for each of n values, from one for each block of the last axis."""
    return scales.repeat_interleave(BLOCK, -1)[..., :n]


def _run_matmul(s):
    k, n = s["case"]["k"], s["case"]["n"]
    a = s["a"].float() * _spread(s["a_scales"], k)
    b = s["b"].float() * _spread(s["b_scales"], k).repeat_interleave(BLOCK, 0)[:n]
    d = torch.matmul(a, b.t())
    if s["bias"] is not None:
        d = d + s["bias"].float()
    return dict(d=d.to(s["d"].dtype))


def _run_grouped(s):
    case, total = s["case"], s["total"]
    experts, k, n = case["experts"], case["k"], case["n"]
    i = torch.arange(total, device="cuda")
    start = s["group_start"].long()
    e = torch.searchsorted(start[1:], i, right=True)
    a = s["a"].float() * _spread(s["a_scales"], k)
    a = a[s["a_rows"][:total].long()] if s["a_rows"] is not None else a[:total]
    rows = torch.zeros(experts, s["most"], k, device="cuda")  # every expert's, padded to the longest
    rows[e, i - start[e]] = a
    b = s["b"].float() * _spread(s["b_scales"], k).repeat_interleave(BLOCK, 1)[:, :n]
    d = torch.bmm(b, rows.transpose(1, 2).contiguous())
    out = torch.zeros_like(s["d"])
    out[:total] = d.transpose(1, 2)[e, i - start[e]].to(out.dtype)
    return dict(d=out)


def _run_combine(s):
    slots = s["slots"].long()
    w = torch.where(slots >= 0, s["weights"], 0.0).unsqueeze(-1)
    return dict(out=(s["x"][slots.clamp(min=0)].float() * w).sum(1).to(s["out"].dtype))


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}.get(case.get("dtype"), 0)
    if case["family"] == "plan":
        return {"bytes": 4 * (3 * case["tokens"] * case["active"] + case["experts"] + 1), "flops": 0}
    if case["family"] == "quantize":
        rows, k = case["rows"], case["columns"]
        return {"bytes": rows * (k * (size * (2 if case["gated"] else 1) + 1) + 4 * _blocks(k)), "flops": 0}
    if case["family"] == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * k + 4 * (m + _blocks(n)) * _blocks(k) + size * n * (m + case["bias"]), "flops": 2 * m * n * k}
    if case["family"] == "grouped":
        sizes, n, k = _group_sizes(case), case["n"], case["k"]
        total, used = sum(sizes), sum(x > 0 for x in sizes)
        rows = min(total, case["tokens"]) if case["gather"] else total
        return {"bytes": rows * (k + 4 * _blocks(k)) + used * (n * k + 4 * _blocks(n) * _blocks(k)) + total * (size * n + 4 * case["gather"]) +
                4 * (case["experts"] + 1), "flops": 2 * total * n * k}
    rows = int(case["tokens"] * case["active"] * case["kept"])
    return {"bytes": size * case["width"] * (rows + case["tokens"]) + 8 * case["tokens"] * case["active"], "flops": 2 * rows * case["width"]}


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    if case["family"] == "plan":
        return None
    if case["family"] == "quantize":
        x, k = s["x"].double(), case["columns"]
        if case["gated"]:
            x = x[:, :k] * x[:, k:] * torch.sigmoid(x[:, k:])
        codes, scales = torch.empty_like(x), torch.empty(case["rows"], _blocks(k), dtype=torch.float64, device="cuda")
        for b in range(_blocks(k)):
            part = x[:, b * BLOCK:(b + 1) * BLOCK]
            scales[:, b] = torch.clamp(part.abs().max(1).values / LARGEST, min=SMALLEST_SCALE)
            codes[:, b * BLOCK:(b + 1) * BLOCK] = part / scales[:, b, None]
        return dict(codes=codes, scales=scales)
    if case["family"] == "combine":
        out = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device="cuda")
        for j in range(case["active"]):
            here = s["slots"][:, j] >= 0
            out[here] += s["weights"][here, j].double().unsqueeze(1) * s["x"][s["slots"][here, j].long()].double()
        return dict(out=out)

    def product(a, a_scales, b, b_scales):
        """Block by block of the inner axis."""
        row = torch.arange(b.shape[0], device="cuda") // BLOCK
        d = torch.zeros(a.shape[0], b.shape[0], dtype=torch.float64, device="cuda")
        for i in range(b_scales.shape[1]):
            at = slice(i * BLOCK, (i + 1) * BLOCK)
            d += (a[:, at].double() @ b[:, at].double().t()) * a_scales[:, i].double()[:, None] * b_scales[:, i].double()[row][None, :]
        return d

    if case["family"] == "matmul":
        d = product(s["a"], s["a_scales"], s["b"], s["b_scales"])
        return dict(d=d if s["bias"] is None else d + s["bias"].double())
    out = torch.zeros(s["d"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for e, count in enumerate(_group_sizes(case)):
        at = s["a_rows"][first:first + count].long() if case["gather"] else torch.arange(first, first + count, device="cuda")
        a = s["a"].view(torch.uint8)[at].view(F8) if s["a"].is_contiguous() else s["a"].float()[at]
        out[first:first + count] = product(a, s["a_scales"][at], s["b"][e], s["b_scales"][e])
        first += count
    return dict(d=out)
