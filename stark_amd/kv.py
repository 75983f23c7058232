"""4-bit paged key/value cache and attention over it, through libstark_qmm (no counterpart in the reference, whose
caches hold 16-bit rows of one session): the calls of a serving loop's step.

    plan = KvPlan(cached, added, free_pages, free_count, block_table, page_size, token_capacity)
    append = KvAppend(cache, k, v, plan.slots, q=q, q_out=q, rotary=Rotary(table, plan.positions))    # per layer
    attend = KvAttention(cache, q, out, block_table, plan.query_start, plan.kv_lengths, max_query, max_kv)
    plan.encode(); append.encode(); attend.encode()

Arguments are marshalled once, when an operator is made: it keeps the tensors it was given, and every encode() reads
what they hold then. encode() is asynchronous on its stream (the current one by default) and may be captured in a
graph. Tensors are GPU tensors; errors are MatmulError with the library's status.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence

import torch

from . import qmm as Q

OUT_OF_PAGES, TABLE_FULL, BAD_LENGTH, TOO_MANY_TOKENS = 1, 2, 4, 8


class _Cache(C.Structure):
    _fields_ = [("data", C.c_void_p), ("data_size", C.c_uint64), ("page_count", C.c_uint32), ("page_size", C.c_uint32),
                ("kv_heads", C.c_uint32), ("head_dim", C.c_uint32), ("group_size", C.c_uint32)]


class _PlanArgs(C.Structure):
    _fields_ = [("struct_size", C.c_uint32)] + [(n, C.c_void_p) for n in (
        "cached", "added", "free_pages", "free_count", "block_table", "query_start", "kv_lengths", "slots", "positions",
        "free_left", "status")] + [(n, C.c_uint32) for n in (
            "batch", "token_capacity", "free_capacity", "table_stride", "page_size")]


class _Rotary(C.Structure):
    _fields_ = [("table", C.c_void_p), ("positions", C.c_void_p), ("position_stride", C.c_uint64),
                ("table_rows", C.c_uint32), ("rotary_dim", C.c_uint32), ("axes", C.c_uint32),
                ("interleaved", C.c_uint32), ("axis_of_pair", C.c_uint8 * 128)]


class _AppendArgs(C.Structure):
    _fields_ = [("struct_size", C.c_uint32), ("cache", _Cache), ("data_type", C.c_uint32)] + [
        (n, C.c_void_p) for n in ("q", "q_out", "k", "v", "slots")] + [
        (n, C.c_uint64) for n in ("q_token_stride", "q_head_stride", "q_out_token_stride", "q_out_head_stride",
                                  "k_token_stride", "k_head_stride", "v_token_stride", "v_head_stride")] + [
        ("tokens", C.c_uint32), ("heads", C.c_uint32), ("rotary", _Rotary)]


class _ReadArgs(C.Structure):
    _fields_ = [("struct_size", C.c_uint32), ("cache", _Cache), ("slots", C.c_void_p), ("data_type", C.c_uint32),
                ("k", C.c_void_p), ("v", C.c_void_p)] + [
        (n, C.c_uint64) for n in ("k_token_stride", "k_head_stride", "v_token_stride", "v_head_stride")] + [
        ("tokens", C.c_uint32)]


class _AttentionArgs(C.Structure):
    _fields_ = [("struct_size", C.c_uint32), ("cache", _Cache), ("data_type", C.c_uint32), ("q", C.c_void_p),
                ("out", C.c_void_p), ("lse", C.c_void_p)] + [
        (n, C.c_uint64) for n in ("q_token_stride", "q_head_stride", "out_token_stride", "out_head_stride")] + [
        (n, C.c_void_p) for n in ("block_table", "query_start", "kv_lengths")] + [
        (n, C.c_uint32) for n in ("batch", "tokens", "heads", "table_stride", "max_query", "max_kv")] + [
        ("scale", C.c_float), ("soft_cap", C.c_float), ("causal", C.c_uint32), ("window", C.c_uint32),
        ("workspace", C.c_void_p), ("workspace_size", C.c_uint64)]


_current_device, _current_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream

_DT = {torch.float32: Q.F32, torch.float16: Q.F16, torch.bfloat16: Q.BF16}


def _dtype(t: torch.Tensor) -> int:
    if t.dtype not in _DT:
        raise Q.MatmulError(Q.UNSUPPORTED_DATA_TYPE, f"{t.dtype}")
    return _DT[t.dtype]


def _require(ok: bool, what: str):
    if not ok:
        raise Q.MatmulError(Q.INVALID_ARGUMENT, what)


def _ints(t: torch.Tensor, count: int, what: str) -> torch.Tensor:
    _require(t.dtype == torch.int32 and t.is_contiguous() and t.numel() >= count, f"{what}: int32, contiguous, {count} or more")
    return t


def _rows(t: Optional[torch.Tensor], tokens: int, heads: int, dim: int, what: str):
    """Pointer and strides of [tokens, heads, dim] rows whose values are contiguous."""
    _require(tuple(t.shape) == (tokens, heads, dim), f"{what}: {tuple(t.shape)} is not {(tokens, heads, dim)}")
    _require(t.stride(2) == 1, f"{what}: the values of a head must be contiguous")
    return Q._ptr(t), t.stride(0), t.stride(1)


class _Operator:
    """Arguments of one call, marshalled; keeps its tensors, which are all on one device."""
    _entry = ""

    def _keep(self, *tensors):
        self._tensors = [t for t in tensors if t is not None]
        for t in self._tensors:
            Q._ptr(t)  # GPU tensors only
        devices = {t.device for t in self._tensors}
        _require(len(devices) == 1, f"{type(self).__name__}: tensors on {sorted(map(str, devices))}")
        self.device = devices.pop()

    def _begin(self, args):
        args.struct_size = C.sizeof(args)
        self._args = args
        self._address = C.addressof(args)
        self._call = getattr(Q.lib(), self._entry)
        self._index = self.device.index

    def encode(self, stream=None) -> None:
        # (torch's own accessors of the current device and stream without their wrappers: 2 us less a call)
        if _current_device() == self._index:
            status = self._call(self._address, _current_stream(self._index) if stream is None else Q._stream(stream))
        else:
            with torch.cuda.device(self.device):
                status = self._call(self._address, _current_stream(self._index) if stream is None else Q._stream(stream))
        if status != Q.OK:
            raise Q.MatmulError(status, type(self).__name__)


class KvCache:
    """One layer's cache (stark_qmm_kv_cache): its memory and geometry."""

    def __init__(self, page_count: int, page_size: int, kv_heads: int, head_dim: int, group_size: int = 64,
                 device="cuda"):
        self.raw = _Cache(None, 0, page_count, page_size, kv_heads, head_dim, group_size)
        size = C.c_uint64()
        Q._check(Q.lib().stark_qmm_kv_cache_size(C.byref(self.raw), C.byref(size)), "KvCache")
        self.data = torch.zeros(size.value, dtype=torch.uint8, device=device)
        self.raw.data, self.raw.data_size = Q._ptr(self.data), size.value
        self.page_count, self.page_size, self.kv_heads = page_count, page_size, kv_heads
        self.head_dim, self.group_size = head_dim, group_size


class KvPlan(_Operator):
    """stark_qmm_kv_plan: block table entries, slots and positions of a step's new tokens from request lengths.
    block_table is written in place; query_start, kv_lengths, slots, positions, free_left and status (OUT_OF_PAGES |
    TABLE_FULL | BAD_LENGTH | TOO_MANY_TOKENS) are made here and rewritten by every encode()."""
    _entry = "stark_qmm_kv_plan"

    def __init__(self, cached: torch.Tensor, added: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
                 block_table: torch.Tensor, page_size: int, token_capacity: int):
        batch = cached.numel()
        _require(block_table.dim() == 2 and block_table.shape[0] == batch, "block_table: [batch, pages]")

        def new(n):
            return torch.empty(n, dtype=torch.int32, device=cached.device)

        self.block_table = block_table
        self.query_start, self.kv_lengths = new(batch + 1), new(batch)
        self.slots, self.positions = new(token_capacity), new(token_capacity)
        self.free_left, self.status = new(1), new(1)
        self._keep(cached, added, free_pages, free_count, block_table, self.query_start, self.kv_lengths, self.slots,
                   self.positions, self.free_left, self.status)
        s = _PlanArgs()
        s.cached, s.added = Q._ptr(_ints(cached, batch, "cached")), Q._ptr(_ints(added, batch, "added"))
        s.free_pages = Q._ptr(_ints(free_pages, 0, "free_pages"))
        s.free_count = Q._ptr(_ints(free_count, 1, "free_count"))
        s.block_table = Q._ptr(_ints(block_table, 0, "block_table"))
        for n in ("query_start", "kv_lengths", "slots", "positions", "free_left", "status"):
            setattr(s, n, Q._ptr(getattr(self, n)))
        s.batch, s.token_capacity, s.free_capacity = batch, token_capacity, free_pages.numel()
        s.table_stride, s.page_size = block_table.shape[1], page_size
        self._begin(s)


class Rotary:
    """stark_qmm_rotary: table [rows, rotary_dim / 2, 2] f32 of (cos, sin), positions int32 [tokens] or [axes, tokens],
    and for several axes the axis that turns each pair."""

    def __init__(self, table: torch.Tensor, positions: torch.Tensor, axis_of_pair: Optional[Sequence[int]] = None,
                 interleaved: bool = False):
        _require(table.dtype == torch.float32 and table.is_contiguous() and table.dim() == 3 and table.shape[2] == 2,
                 "table: f32 [rows, pairs, 2]")
        positions = positions if positions.dim() == 2 else positions.view(1, -1)
        _require(positions.dtype == torch.int32 and (positions.shape[1] <= 1 or positions.stride(1) == 1),
                 "positions: int32 [axes, tokens]")
        pairs = table.shape[1]
        axes = [0] * pairs if axis_of_pair is None else list(axis_of_pair)
        _require(len(axes) == pairs and pairs <= 128 and all(0 <= x < 256 for x in axes), "axis_of_pair: one of each pair")
        self.table, self.positions = table, positions
        self.raw = _Rotary(Q._ptr(table), Q._ptr(positions), positions.stride(0), table.shape[0], 2 * pairs,
                           positions.shape[0], int(interleaved))
        for i, x in enumerate(axes):
            self.raw.axis_of_pair[i] = x


class KvAppend(_Operator):
    """stark_qmm_kv_append: rotates query (q to q_out, which may be q) and key rows [tokens, heads, head_dim] and writes
    the keys and values of each token to its slot in 4 bits."""
    _entry = "stark_qmm_kv_append"

    def __init__(self, cache: KvCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
                 q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None, rotary: Optional[Rotary] = None):
        tokens = k.shape[0]
        self.cache, self.rotary = cache, rotary
        self._keep(cache.data, k, v, slots, q, q_out, *((rotary.table, rotary.positions) if rotary else ()))
        _require((q is None) == (q_out is None), "q and q_out go together")
        _require(all(t.dtype == k.dtype for t in (v, q, q_out) if t is not None), "q, k and v are of one type")
        s = _AppendArgs()
        s.cache, s.data_type, s.tokens = cache.raw, _dtype(k), tokens
        s.slots = Q._ptr(_ints(slots, tokens, "slots"))
        s.k, s.k_token_stride, s.k_head_stride = _rows(k, tokens, cache.kv_heads, cache.head_dim, "k")
        s.v, s.v_token_stride, s.v_head_stride = _rows(v, tokens, cache.kv_heads, cache.head_dim, "v")
        if q is not None:
            s.heads = q.shape[1]
            s.q, s.q_token_stride, s.q_head_stride = _rows(q, tokens, s.heads, cache.head_dim, "q")
            s.q_out, s.q_out_token_stride, s.q_out_head_stride = _rows(q_out, tokens, s.heads, cache.head_dim, "q_out")
        if rotary is not None:
            _require(rotary.positions.shape[1] >= tokens, "positions: one of each token")
            s.rotary = rotary.raw
        self._begin(s)


class KvRead(_Operator):
    """stark_qmm_kv_read: rows at the slots as the values that their 4 bits stand for, into k and v (either may be None)."""
    _entry = "stark_qmm_kv_read"

    def __init__(self, cache: KvCache, slots: torch.Tensor, k: Optional[torch.Tensor], v: Optional[torch.Tensor]):
        some = k if k is not None else v
        _require(some is not None and (k is None or v is None or k.dtype == v.dtype), "k or v, of one type")
        tokens = some.shape[0]
        self.cache = cache
        self._keep(cache.data, slots, k, v)
        s = _ReadArgs()
        s.cache, s.data_type, s.tokens = cache.raw, _dtype(some), tokens
        s.slots = Q._ptr(_ints(slots, tokens, "slots"))
        if k is not None:
            s.k, s.k_token_stride, s.k_head_stride = _rows(k, tokens, cache.kv_heads, cache.head_dim, "k")
        if v is not None:
            s.v, s.v_token_stride, s.v_head_stride = _rows(v, tokens, cache.kv_heads, cache.head_dim, "v")
        self._begin(s)


class KvAttention(_Operator):
    """stark_qmm_kv_attention: out = softmax(scale q k^T) v over the cache, scale 1 / sqrt(head_dim) by default; q and out
    [tokens, heads, head_dim] in f16 or bf16, lse [tokens, heads] f32 if given. max_query and max_kv bound the lengths
    of any request in any encode(). The workspace is made here unless one is given; operators whose encode() calls may
    overlap (two streams, two captured graphs) must not share one."""
    _entry = "stark_qmm_kv_attention"

    def __init__(self, cache: KvCache, q: torch.Tensor, out: torch.Tensor, block_table: torch.Tensor,
                 query_start: torch.Tensor, kv_lengths: torch.Tensor, max_query: int, max_kv: int,
                 scale: Optional[float] = None, causal: bool = True, window: int = 0, soft_cap: float = 0.0,
                 lse: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None):
        _require(block_table.dim() == 2, "block_table: [batch, pages]")
        tokens, heads, batch = q.shape[0], q.shape[1], block_table.shape[0]
        self.cache, self.out, self.lse = cache, out, lse
        self._keep(cache.data, q, out, block_table, query_start, kv_lengths, lse, workspace)
        _require(out.dtype == q.dtype, "q and out are of one type")
        _require(lse is None or (lse.dtype == torch.float32 and lse.is_contiguous() and lse.numel() == tokens * heads),
                 "lse: f32 [tokens, heads]")
        s = _AttentionArgs()
        s.cache, s.data_type, s.lse = cache.raw, _dtype(q), Q._ptr(lse)
        s.q, s.q_token_stride, s.q_head_stride = _rows(q, tokens, heads, cache.head_dim, "q")
        s.out, s.out_token_stride, s.out_head_stride = _rows(out, tokens, heads, cache.head_dim, "out")
        s.block_table = Q._ptr(_ints(block_table, 0, "block_table"))
        s.query_start = Q._ptr(_ints(query_start, batch + 1, "query_start"))
        s.kv_lengths = Q._ptr(_ints(kv_lengths, batch, "kv_lengths"))
        s.batch, s.tokens, s.heads, s.table_stride = batch, tokens, heads, block_table.shape[1]
        s.max_query, s.max_kv = max_query, max_kv
        s.scale = 1.0 / math.sqrt(cache.head_dim) if scale is None else scale
        s.soft_cap, s.causal, s.window = soft_cap, int(causal), window
        need = C.c_uint64()
        s.struct_size = C.sizeof(s)
        with torch.cuda.device(q.device):  # its size depends on the device's compute units
            Q._check(Q.lib().stark_qmm_kv_attention_workspace_size(C.byref(s), C.byref(need)), "KvAttention")
        self.workspace_bytes = need.value
        if workspace is None and need.value:
            workspace = torch.empty(need.value, dtype=torch.uint8, device=q.device)
        if workspace is not None:
            s.workspace, s.workspace_size = Q._ptr(workspace), Q._nbytes(workspace)
        self.workspace = workspace
        self._begin(s)
