"""Products of 8-bit floating-point (e4m3) codes with block scales, through libstark_qmm (no counterpart in the reference,
whose 8-bit weights are integers), and what routed experts need around them:

    codes, scales = new_rows(tokens, model)                                                  # dense layer
    quantize = Fp8Quantize(x, codes, scales)
    product = Fp8Matmul(codes, scales, weights, weight_scales, y)

    plan = ExpertPlan(ids.view(tokens, active), experts)                                     # routed experts
    up = Fp8GroupedMatmul(codes, scales, up_w, up_s, h, plan.group_start, a_rows=plan.tokens)
    gate = Fp8Quantize(h, h_codes, h_scales, gated=True, row_count=plan.count)
    down = Fp8GroupedMatmul(h_codes, h_scales, down_w, down_s, r, plan.group_start)
    combine = ExpertCombine(r, plan.slots, weights, out)

Codes are torch.float8_e4m3fn or uint8 tensors whose rows start on 16-byte boundaries, scales float32: one for each row and
128 values of activations, one for each 128 x 128 values of weights. Arguments are marshalled once, when an operator is made:
it keeps the tensors it was given, and every encode() reads what they hold then. encode() is asynchronous on its stream (the
current one by default) and may be captured in a graph. An operator outlives the graphs that hold its calls, and its calls on a
stream that is given as a bare handle. Tensors are GPU tensors; errors are MatmulError with the library's status.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import qmm as Q
from .kv import _Operator, _dtype, _ints, _require

BLOCK = 128
_CODES = (torch.float8_e4m3fn, torch.uint8)


class _QuantizeArgs(C.Structure):
    _fields_ = [("struct_size", C.c_uint32), ("data_type", C.c_uint32), ("x", C.c_void_p), ("x_row_stride", C.c_uint64),
                ("codes", C.c_void_p), ("code_row_stride", C.c_uint64), ("scales", C.c_void_p),
                ("scale_row_stride", C.c_uint64), ("scale_block_stride", C.c_uint64), ("rows", C.c_uint32),
                ("columns", C.c_uint32), ("gated", C.c_uint32), ("row_count", C.c_void_p)]


class _MatmulArgs(C.Structure):
    _fields_ = [("struct_size", C.c_uint32), ("d_type", C.c_uint32), ("a", C.c_void_p), ("a_row_stride", C.c_uint64),
                ("a_scales", C.c_void_p), ("a_scale_row_stride", C.c_uint64), ("a_scale_block_stride", C.c_uint64),
                ("b", C.c_void_p), ("b_row_stride", C.c_uint64), ("b_scales", C.c_void_p),
                ("b_scale_row_stride", C.c_uint64), ("b_scale_block_stride", C.c_uint64), ("d", C.c_void_p),
                ("d_row_stride", C.c_uint64), ("d_ops", Q._DOps), ("m", C.c_uint32), ("n", C.c_uint32), ("k", C.c_uint32),
                ("workspace", C.c_void_p), ("workspace_size", C.c_uint64)]


class _GroupedArgs(C.Structure):
    _fields_ = [("struct_size", C.c_uint32), ("product", _MatmulArgs), ("experts", C.c_uint32), ("group_start", C.c_void_p),
                ("b_expert_stride", C.c_uint64), ("b_scale_expert_stride", C.c_uint64), ("bias_expert_stride", C.c_uint64),
                ("a_rows", C.c_void_p), ("a_row_count", C.c_uint32)]


class _PlanArgs(C.Structure):
    _fields_ = [("struct_size", C.c_uint32)] + [(n, C.c_void_p) for n in ("ids", "group_start", "tokens_out", "slots")] + [
        (n, C.c_uint32) for n in ("tokens", "active", "experts", "first")] + [
        ("workspace", C.c_void_p), ("workspace_size", C.c_uint64)]


class _CombineArgs(C.Structure):
    _fields_ = [("struct_size", C.c_uint32), ("data_type", C.c_uint32)] + [
        (n, C.c_void_p) for n in ("x", "slots", "weights", "out")] + [
        ("x_row_stride", C.c_uint64), ("out_row_stride", C.c_uint64)] + [
        (n, C.c_uint32) for n in ("tokens", "active", "rows", "width", "accumulate")]


def blocks(n: int) -> int:
    return -(-n // BLOCK)


def new_rows(rows: int, columns: int, device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes [rows, columns] (e4m3, rows on 16-byte boundaries) and scales [rows, blocks] for Fp8Quantize to fill."""
    codes = torch.zeros(rows, -(-columns // 16) * 16, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)[:, :columns]
    return codes, torch.zeros(rows, blocks(columns), dtype=torch.float32, device=device)


def _counts(what: str, *n: int):
    """Sizes that the library's 32 bits hold (its own limits are lower; ctypes would cut what is above)."""
    _require(all(0 <= x < 1 << 32 for x in n), f"{what}: {n} are no sizes")


def _matrix(t: torch.Tensor, rows: int, columns: int, what: str):
    """Pointer and row stride of [rows, columns] whose rows are contiguous."""
    _counts(what, rows, columns)
    _require(tuple(t.shape) == (rows, columns), f"{what}: {tuple(t.shape)} is not {(rows, columns)}")
    _require(columns <= 1 or t.stride(1) == 1 or t.numel() == 0, f"{what}: the values of a row must be contiguous")
    return Q._ptr(t), t.stride(0) if rows > 1 else columns


def _codes(t: torch.Tensor, what: str):
    """Pointer and row stride of rows of codes, which may be read up to the next 16-byte boundary."""
    _require(t.dtype in _CODES, f"{what}: float8_e4m3fn or uint8")
    rows, columns = t.shape[-2], t.shape[-1]
    ptr, stride = _matrix(t if t.dim() == 2 else t[0], rows, columns, what)
    last = sum((n - 1) * s for n, s in zip(t.shape[:-1], t.stride()[:-1])) + -(-columns // 16) * 16
    _require(t.numel() == 0 or t.storage_offset() + last <= t.untyped_storage().nbytes(),
             f"{what}: the last row's memory ends before a 16-byte boundary")
    return ptr, stride


def _scales(t: torch.Tensor, rows: int, count: int, what: str):
    """Pointer and strides of [rows, blocks] scales."""
    _require(t.dtype == torch.float32 and tuple(t.shape) == (rows, count), f"{what}: f32 {(rows, count)}, not {t.dtype} {tuple(t.shape)}")
    return Q._ptr(t), t.stride(0), t.stride(1)


class Fp8Quantize(_Operator):
    """stark_qmm_fp8_quantize: rows x [rows, columns] (gated: [rows, 2 * columns], of value * silu(gate)) to e4m3 codes and a
    scale for each 128 values. row_count: int32 on the device, the rows to take."""
    _entry = "stark_qmm_fp8_quantize"

    def __init__(self, x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, gated: bool = False,
                 row_count: Optional[torch.Tensor] = None):
        _require(codes.dim() == 2 and x.dim() == 2, "x and codes: [rows, columns]")
        rows, columns = codes.shape
        self._keep(x, codes, scales, row_count)
        s = _QuantizeArgs()
        s.data_type, s.rows, s.columns, s.gated = _dtype(x), rows, columns, int(gated)
        s.x, s.x_row_stride = _matrix(x, rows, columns * (2 if gated else 1), "x")
        _require(codes.dtype in _CODES, "codes: float8_e4m3fn or uint8")
        s.codes, s.code_row_stride = _matrix(codes, rows, columns, "codes")
        s.scales, s.scale_row_stride, s.scale_block_stride = _scales(scales, rows, blocks(columns), "scales")
        if row_count is not None:
            s.row_count = Q._ptr(_ints(row_count, 1, "row_count"))
        self.codes, self.scales = codes, scales
        self._begin(s)


class _Product(_Operator):
    def _product(self, a, a_scales, b, b_scales, d, m, a_count, bias, ab_scale, accumulate, soft_cap):
        """The arguments that both products have; b, b_scales and bias of the first expert."""
        _require(a.dim() == 2 and d.dim() == 2, "a: [rows, k], d: [m, n]")
        (n, k), out = b.shape, _MatmulArgs()
        _require(a.shape[1] == k, f"a and b: k is {a.shape[1]} and {k}")
        out.struct_size = C.sizeof(out)
        out.d_type, out.m, out.n, out.k = _dtype(d), m, n, k
        _require(a.shape[0] == a_count, f"a: {a.shape[0]} rows, not {a_count}")
        out.a, out.a_row_stride = _codes(a, "a")
        out.a_scales, out.a_scale_row_stride, out.a_scale_block_stride = _scales(a_scales, a_count, blocks(k), "a_scales")
        out.b, out.b_row_stride = _codes(b, "b")
        out.b_scales, out.b_scale_row_stride, out.b_scale_block_stride = _scales(b_scales, blocks(n), blocks(k), "b_scales")
        out.d, out.d_row_stride = _matrix(d, m, n, "d")
        if bias is not None:
            _require(bias.dtype == d.dtype and tuple(bias.shape) == (n,) and (n <= 1 or bias.stride(0) == 1),
                     "bias: [n] in d's type")
            out.d_ops.bias = Q._ptr(bias)
        out.d_ops.ab_scale, out.d_ops.accumulate = ab_scale, int(accumulate)
        out.d_ops.has_soft_cap, out.d_ops.soft_cap = int(soft_cap is not None), soft_cap or 0.0
        return out

    def _space(self, args, product, workspace):
        """The workspace that the call needs, made here unless one is given."""
        need = C.c_uint64()
        args.struct_size = C.sizeof(args)
        with torch.cuda.device(self.device):
            Q._check(getattr(Q.lib(), self._entry + "_workspace_size")(C.byref(args), C.byref(need)), type(self).__name__)
        self.workspace_bytes = need.value
        if workspace is None and need.value:
            workspace = torch.empty(need.value, dtype=torch.uint8, device=self.device)
            self._make(workspace)
        if workspace is not None:
            product.workspace, product.workspace_size = Q._ptr(workspace), Q._nbytes(workspace)
        self.workspace = workspace


class Fp8Matmul(_Product):
    """stark_qmm_fp8_matmul: d [m, n] (f32, f16 or bf16) = ab_scale * a b^T of codes a [m, k] and b [n, k] with a_scales
    [m, blocks] and b_scales [blocks, blocks], plus d if accumulate, plus bias [n]; then soft_cap * tanh(. / soft_cap).
    Operators whose encode() calls may overlap (two streams, two captured graphs) must not share a workspace."""
    _entry = "stark_qmm_fp8_matmul"

    def __init__(self, a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor, d: torch.Tensor,
                 bias: Optional[torch.Tensor] = None, ab_scale: float = 1.0, accumulate: bool = False,
                 soft_cap: Optional[float] = None, workspace: Optional[torch.Tensor] = None):
        _require(b.dim() == 2, "b: [n, k]")
        self._keep(a, a_scales, b, b_scales, d, bias, workspace)
        s = self._product(a, a_scales, b, b_scales, d, d.shape[0], d.shape[0], bias, ab_scale, accumulate, soft_cap)
        self._space(s, s, workspace)
        self.d = d
        self._begin(s)


class Fp8GroupedMatmul(_Product):
    """stark_qmm_fp8_grouped_matmul: rows group_start[e] .. group_start[e + 1] - 1 of d [m, n] from expert e's matrix of b
    [experts, n, k], b_scales [experts, blocks, blocks] and bias [experts, n]; row i from row a_rows[i] of a, or row i.
    Rows that no group has stay as they were."""
    _entry = "stark_qmm_fp8_grouped_matmul"

    def __init__(self, a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor, d: torch.Tensor,
                 group_start: torch.Tensor, a_rows: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                 ab_scale: float = 1.0, accumulate: bool = False, soft_cap: Optional[float] = None,
                 workspace: Optional[torch.Tensor] = None):
        _require(b.dim() == 3 and b_scales.dim() == 3 and b.shape[0] == b_scales.shape[0] > 0, "b, b_scales: [experts, ...]")
        _require(bias is None or (bias.dim() == 2 and bias.shape[0] == b.shape[0]), "bias: [experts, n]")
        self._keep(a, a_scales, b, b_scales, d, group_start, a_rows, bias, workspace)
        _codes(b, "b")
        _counts("experts", b.shape[0])
        s, m = _GroupedArgs(), d.shape[0]
        s.product = self._product(a, a_scales, b[0], b_scales[0], d, m, a.shape[0] if a_rows is not None else m,
                                  None if bias is None else bias[0], ab_scale, accumulate, soft_cap)
        s.experts = b.shape[0]
        s.group_start = Q._ptr(_ints(group_start, s.experts + 1, "group_start"))
        s.b_expert_stride, s.b_scale_expert_stride = b.stride(0), b_scales.stride(0)
        s.bias_expert_stride = bias.stride(0) if bias is not None else 0
        if a_rows is not None:
            s.a_rows, s.a_row_count = Q._ptr(_ints(a_rows, m, "a_rows")), a.shape[0]
        self._space(s, s.product, workspace)
        self.d = d
        self._begin(s)


class ExpertPlan(_Operator):
    """stark_qmm_expert_plan: routes ids [tokens, active] (int32; moe_route's, which are flat, as a view) in the order of the experts
    first .. first + experts - 1. group_start [experts + 1], tokens [tokens * active] (-1 behind the last) and slots [tokens,
    active] (-1: another's expert) are made here and rewritten by every encode(); count is group_start's last."""
    _entry = "stark_qmm_expert_plan"

    def __init__(self, ids: torch.Tensor, experts: int, first: int = 0, workspace: Optional[torch.Tensor] = None):
        _require(ids.dim() == 2 and ids.dtype == torch.int32 and ids.is_contiguous(), "ids: int32 [tokens, active], contiguous")
        _require(experts >= 1 and first >= 0, "experts: 1 or more, from 0 on")
        _counts("ids, experts and the first", *ids.shape, experts, first)

        def new(*n):
            return torch.empty(*n, dtype=torch.int32, device=ids.device)

        self.group_start, self.tokens, self.slots = new(experts + 1), new(ids.numel()), new(*ids.shape)
        self.count = self.group_start[experts:]
        self._keep(ids, self.group_start, self.tokens, self.slots, workspace)
        self._make(self.group_start, self.tokens, self.slots)
        s = _PlanArgs()
        s.struct_size = C.sizeof(s)
        s.ids, s.group_start, s.tokens_out, s.slots = (Q._ptr(t) for t in (ids, self.group_start, self.tokens, self.slots))
        s.tokens, s.active, s.experts, s.first = ids.shape[0], ids.shape[1], experts, first
        need = C.c_uint64()
        Q._check(Q.lib().stark_qmm_expert_plan_workspace_size(C.byref(s), C.byref(need)), "ExpertPlan")
        self.workspace_bytes = need.value
        if workspace is None and need.value:
            workspace = torch.empty(need.value, dtype=torch.uint8, device=ids.device)
            self._make(workspace)
        if workspace is not None:
            s.workspace, s.workspace_size = Q._ptr(workspace), Q._nbytes(workspace)
        self.workspace = workspace
        self._begin(s)


class ExpertCombine(_Operator):
    """stark_qmm_expert_combine: out [tokens, width] = (out if accumulate) + sum over j of weights[t, j] * x[slots[t, j]];
    slots outside x's rows are not counted."""
    _entry = "stark_qmm_expert_combine"

    def __init__(self, x: torch.Tensor, slots: torch.Tensor, weights: torch.Tensor, out: torch.Tensor, accumulate: bool = False):
        _require(x.dim() == 2 and out.dim() == 2 and slots.dim() == 2, "x, out, slots: two axes")
        (tokens, active), (rows, width) = slots.shape, x.shape
        _counts("slots", tokens, active)
        self._keep(x, slots, weights, out)
        _require(x.dtype == out.dtype, "x and out are of one type")
        _require(weights.dtype == torch.float32 and weights.is_contiguous() and weights.numel() == tokens * active,
                 "weights: f32 [tokens, active]")
        s = _CombineArgs()
        s.data_type, s.tokens, s.active, s.rows, s.width, s.accumulate = _dtype(x), tokens, active, rows, width, int(accumulate)
        s.x, s.x_row_stride = _matrix(x, rows, width, "x")
        s.out, s.out_row_stride = _matrix(out, tokens, width, "out")
        s.slots, s.weights = Q._ptr(_ints(slots, tokens * active, "slots")), Q._ptr(weights)
        self.out = out
        self._begin(s)
