"""Token-transformer operators over the C ABI of include/musev_tokens.h: packed attention, rotary positions with several axes, the gated
residual norm and the int8 projection.  They are part of :mod:`musev_amd.ops` (``from musev_amd import ops; ops.attention_packed(...)``)
and follow its manner: 2-D row matrices with unit inner stride, no CPU path, launches on the current stream of the tensors' device.
fp16 and bf16; forward only, like the rest of the framework.

Each call reads its tensors on the stream it is made on: a tensor made on another stream has to be finished there first.  Nothing is kept
between calls; what a call needs besides its arguments is allocated for that call (inside a graph capture: from the capture's pool), so
concurrent calls and several captured graphs never share it.  A graph refers to the plan, table or codes it was captured with: keep them.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import List, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from ._lib import MV_ACT_NONE, MV_ACT_SILU, AttnPackedDesc, GatedNormDesc, GemmI8Desc, RotaryDesc, check

__all__ = ["AttentionPlan", "attention_plan", "attention_packed", "RotaryTable", "rotary_table", "rotary_axes", "gated_residual_norm",
           "Int8Rows", "pack_weight_i8", "quantize_rows_i8", "gemm_i8", "linear_i8"]

_DTYPES = {torch.float16: 0, torch.bfloat16: 1}
_I32_MAX = 2 ** 31 - 1


def _on_gpu(t: torch.Tensor) -> bool:
    return t.is_cuda


class _device_of:
    """makes ``dev`` the current device for a launch (only where it is not already) and gives the raw handle of its current stream"""

    def __init__(self, dev: torch.device):
        self.idx = dev.index

    def __enter__(self) -> int:
        self.prev = torch.cuda.current_device()
        if self.prev != self.idx:
            torch.cuda.set_device(self.idx)
        return torch.cuda.current_stream(self.idx).cuda_stream

    def __exit__(self, *exc) -> None:
        if self.prev != self.idx:
            torch.cuda.set_device(self.prev)


def _matrix(t: torch.Tensor, name: str, dtype: Optional[torch.dtype] = None, device: Optional[torch.device] = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{name}: expected a 2-D tensor with unit inner stride, got "
                         f"{(tuple(t.shape), t.stride()) if isinstance(t, torch.Tensor) else type(t).__name__}")
    if not _on_gpu(t) or (t.dtype not in _DTYPES if dtype is None else t.dtype != dtype):
        raise ValueError(f"{name}: expected a CUDA {'fp16 | bf16' if dtype is None else dtype} tensor, got {t.dtype} on {t.device}")
    if device is not None and t.device != device:
        raise ValueError(f"{name}: on {t.device}, the other tensors are on {device}")
    if t.shape[0] > 1 and (t.stride(0) > _I32_MAX or (t.stride(0) < t.shape[1])):
        raise ValueError(f"{name}: row stride {t.stride(0)} for {t.shape[1]} columns")
    return t


def _ld(t: torch.Tensor) -> int:
    """row stride in elements (a single row has none of its own)"""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _span(t: torch.Tensor) -> Tuple[int, int]:
    if t.numel() == 0:
        return 0, 0
    return t.data_ptr(), t.data_ptr() + ((t.shape[0] - 1) * _ld(t) + t.shape[1]) * t.element_size()


def _columns_apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """two column ranges of one matrix (slices of a fused projection): same row stride, and no column in common"""
    if _ld(a) != _ld(b) or a.element_size() != b.element_size():
        return False
    es, ld = a.element_size(), _ld(a)
    off = (b.data_ptr() - a.data_ptr()) % (ld * es)
    return off >= a.shape[1] * es and off + b.shape[1] * es <= ld * es


def _no_overlap(out: torch.Tensor, name: str, inputs: Sequence[Tuple[str, Optional[torch.Tensor]]], same_ok: Sequence[str] = ()) -> None:
    """an output may be an input itself where the operator reads an element before it writes it (``same_ok``), never part of one"""
    o0, o1 = _span(out)
    for nm, t in inputs:
        if t is None or t.numel() == 0 or o0 == o1:
            continue
        t0, t1 = _span(t) if t.dim() == 2 else (t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
        if t1 <= o0 or o1 <= t0:
            continue
        if nm in same_ok and t0 == o0 and t.shape == out.shape and _ld(t) == _ld(out):
            continue
        if t.dim() == 2 and _columns_apart(t, out):
            continue
        raise ValueError(f"{name}: overlaps {nm}" + (" (it may be the very same matrix)" if nm in same_ok else ""))


class _Held:
    """device memory that belongs to a plan, table or weight: made on one stream, perhaps used on others"""

    def _hold(self, *tensors: torch.Tensor) -> None:
        self._tensors = tensors
        self.device = tensors[0].device
        self._streams = {torch.cuda.current_stream(self.device).cuda_stream} if tensors[0].is_cuda else set()

    def _use(self, stream: int) -> None:
        # the allocator may not hand the memory out again while a launch on another stream still reads it
        if stream not in self._streams and not torch.cuda.is_current_stream_capturing():
            for t in self._tensors:
                t.record_stream(torch.cuda.current_stream(self.device))
            self._streams.add(stream)


# ---- packed attention ---------------------------------------------------------------------------------------------------------
class AttentionPlan(_Held):
    """the work list of :func:`attention_packed` for one set of sequence lengths (:func:`attention_plan`)"""

    def __init__(self, q_lens, kv_lens, heads, kv_heads, d, causal, scale, n_items, n_few, items, joins, ws_rows):
        self.q_lens, self.kv_lens = tuple(q_lens), tuple(kv_lens)
        self.heads, self.kv_heads, self.d, self.causal, self.scale = heads, kv_heads, d, causal, scale
        self.total_q, self.total_kv = sum(q_lens), sum(kv_lens)
        self._hold(items, joins)
        ds = AttnPackedDesc()
        ds.items, ds.joins = items.data_ptr(), joins.data_ptr()
        ds.n_items, ds.n_few, ds.n_joins, ds.ws_rows = n_items, n_few, joins.shape[0], ws_rows
        ds.heads, ds.kv_heads, ds.d, ds.causal, ds.scale = heads, kv_heads, d, int(causal), scale
        self._desc = ds
        self._workspace = 4 * ws_rows * kv_heads * (d + 2)   # mv_attention_packed_workspace_bytes


def _lens(v, name: str) -> List[int]:
    if isinstance(v, torch.Tensor):
        if v.is_cuda:
            raise ValueError(f"{name}: lengths are host integers (reading them from the GPU would wait for it)")
        v = v.tolist()
    v = [int(x) for x in v]
    if not v or min(v) < 0 or sum(v) > _I32_MAX:
        raise ValueError(f"{name}: expected at least one length, none negative, at most 2^31 - 1 rows in all")
    return v


WIDE_ROWS, FEW_ROWS = 128, 32   # packed rows per item of the two kernel forms
# Keys of an item that is worth a split: an item's parts each write and the join reads back (d + 2) fp32 per row.
MIN_PART_WIDE, MIN_PART_FEW = 512, 256
BLOCKS = 512                    # two blocks on each of the 256 CUs


def _plan_items(ql: Sequence[int], kl: Sequence[int], group: int, kv_heads: int, causal: bool):
    """(wide items, few-row items, joins, workspace rows): see include/musev_tokens.h.  A sequence of at most FEW_ROWS packed rows makes one
    few-row item.  An item's keys end with what its last query sees.  Where the items alone would leave CUs idle, or one item would outlast
    the others, its keys are split into parts of about 1 / BLOCKS of all the work; the longest items come first."""
    tiles, q_row, k_row = ([], []), 0, 0
    for q, kv in zip(ql, kl):
        rows = q * group
        few = rows <= FEW_ROWS
        for m0 in range(0, rows, FEW_ROWS if few else WIDE_ROWS):
            last = min(m0 + (FEW_ROWS if few else WIDE_ROWS), rows) - 1
            end = max(0, min(kv, last // group + kv - q + 1)) if causal else kv
            tiles[few].append((q_row, q, k_row, kv, m0, end))
        q_row, k_row = q_row + q, k_row + kv
    out, joins, ws = ([], []), [], 0
    for few in (False, True):
        width, least = (FEW_ROWS, MIN_PART_FEW) if few else (WIDE_ROWS, MIN_PART_WIDE)
        part = max(least, -(-sum(t[5] for t in tiles[few]) * kv_heads // BLOCKS))
        part = -(-part // 64) * 64
        for q_row, q, k_row, kv, m0, end in tiles[few]:
            n = max(1, (end + part // 2) // part)
            if n == 1:
                out[few].append((q_row, q, k_row, kv, m0, 0, end, -1))
                continue
            size = -(-(-(-end // n)) // 64) * 64
            n = -(-end // size)
            rows = min(width, q * group - m0)
            for s in range(n):
                out[few].append((q_row, q, k_row, kv, m0, s * size, min(end, (s + 1) * size), ws + s * rows))
            joins.append((q_row, q, kv, m0, ws, n, rows, 0))
            ws += n * rows
        out[few].sort(key=lambda i: i[5] - i[6])
    return out[0], out[1], joins, ws


def attention_plan(q_lens: Sequence[int], kv_lens: Optional[Sequence[int]] = None, *, heads: int, kv_heads: Optional[int] = None, d: int,
                   causal: bool = True, scale: Optional[float] = None, device: Union[str, torch.device] = "cuda") -> AttentionPlan:
    """The plan of :func:`attention_packed` over ``len(q_lens)`` sequences of ``q_lens[i]`` query and ``kv_lens[i]`` key rows (default: as
    many), host integers, zero allowed.  ``causal``: query i of a sequence sees keys j <= i + kv_len - q_len -- the new tokens stand at the
    end of their keys.  ``scale``: of the scores, default d ** -0.5.  Made once per set of lengths and used for every layer."""
    kv_heads = heads if kv_heads is None else int(kv_heads)
    heads, d = int(heads), int(d)
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"attention_plan: {heads} heads over {kv_heads} key / value heads")
    if d < 8 or d > 128 or d % 8:
        raise ValueError(f"attention_plan: head dim {d} (a multiple of 8 up to 128)")
    ql = _lens(q_lens, "q_lens")
    kl = ql if kv_lens is None else _lens(kv_lens, "kv_lens")
    if len(ql) != len(kl):
        raise ValueError(f"attention_plan: {len(ql)} query and {len(kl)} key lengths")
    if max(ql) * (heads // kv_heads) > _I32_MAX:
        raise ValueError("attention_plan: more than 2^31 - 1 (query, head) rows per key / value head")
    scale = d ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= 1e6:
        raise ValueError(f"attention_plan: scale {scale} (at most 1e6 in size)")
    dev = torch.device(device)
    if dev.type == "cuda" and dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    wide, few, joins, ws_rows = _plan_items(ql, kl, heads // kv_heads, kv_heads, bool(causal))
    # one upload for both tables
    table = torch.tensor((wide + few + joins) or [(0,) * 8], dtype=torch.int32).to(dev)
    n = len(wide) + len(few)
    return AttentionPlan(ql, kl, heads, kv_heads, d, bool(causal), scale, len(wide), len(few), table[:n], table[n:n + len(joins)], ws_rows)


def attention_packed(plan: AttentionPlan, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Softmax attention of packed sequences: ``q`` [>= total_q, heads * d], ``k`` / ``v`` [>= total_kv, kv_heads * d], fp16 or bf16, any row
    stride that keeps rows 16-byte aligned (column slices of a fused projection).  Returns [total_q, heads * d], or writes the first
    total_q rows of ``out`` and leaves the rows behind them as they were.  A query that sees no key gives 0; what a query does not see --
    later tokens, other sequences, rows behind the last one -- does not reach its output, NaN and infinities included."""
    _matrix(q, "q")
    _matrix(k, "k", q.dtype, q.device)
    _matrix(v, "v", q.dtype, q.device)
    hd, kvd = plan.heads * plan.d, plan.kv_heads * plan.d
    if q.shape[1] != hd or q.shape[0] < plan.total_q:
        raise ValueError(f"attention_packed: q {tuple(q.shape)}, the plan has {plan.total_q} rows of {hd}")
    for t, nm in ((k, "k"), (v, "v")):
        if t.shape[1] != kvd or t.shape[0] < plan.total_kv:
            raise ValueError(f"attention_packed: {nm} {tuple(t.shape)}, the plan has {plan.total_kv} rows of {kvd}")
    for t, nm in ((q, "q"), (k, "k"), (v, "v")) + (((_matrix(out, "out", q.dtype, q.device), "out"),) if out is not None else ()):
        if t.data_ptr() % 16 or _ld(t) % 8 or _ld(t) > 1 << 23:
            raise ValueError(f"attention_packed: {nm}: rows must be 16-byte aligned and at most 2^23 elements apart, row stride {_ld(t)}")
    if plan.device != q.device:
        raise ValueError(f"attention_packed: plan on {plan.device}, tensors on {q.device}")
    if out is None:
        out = torch.empty((plan.total_q, hd), dtype=q.dtype, device=q.device)
    else:
        if out.shape[1] != hd or out.shape[0] < plan.total_q:
            raise ValueError(f"attention_packed: out {tuple(out.shape)}, the plan has {plan.total_q} rows of {hd}")
        _no_overlap(out[:plan.total_q], "attention_packed: out", (("q", q), ("k", k), ("v", v)))
    ds = AttnPackedDesc.from_buffer_copy(plan._desc)
    ds.q, ds.k, ds.v, ds.out = q.data_ptr(), k.data_ptr() or q.data_ptr(), v.data_ptr() or q.data_ptr(), out.data_ptr()   # (no key at all: not read)
    ds.ldq, ds.ldk, ds.ldv, ds.ldo, ds.dtype = _ld(q), _ld(k), _ld(v), _ld(out), _DTYPES[q.dtype]
    with _device_of(q.device) as stream:
        plan._use(stream)
        ws = None
        if plan._workspace:
            ws = torch.empty(plan._workspace, dtype=torch.uint8, device=q.device)
            ds.workspace, ds.workspace_bytes = ws.data_ptr(), plan._workspace
        check(_lib.load().mv_attention_packed(C.byref(ds), stream), "mv_attention_packed")
    return out


# ---- rotary positions ----------------------------------------------------------------------------------------------------------
class RotaryTable(_Held):
    """axis and turns per position step of every pair of a head (:func:`rotary_table`)"""

    def __init__(self, turns: torch.Tensor, axis: torch.Tensor, axes: int):
        self.pairs, self.axes = turns.numel(), axes
        self.turns, self.axis = turns, axis
        self._hold(turns, axis)


def rotary_table(sections: Sequence[int], theta: float = 10000.0, *, shared: bool = False, device: Union[str, torch.device] = "cuda") -> RotaryTable:
    """Frequencies of rotary positions with ``len(sections)`` axes: ``sections[a]`` (even) of a head's elements turn with axis a -- for a video
    (time, height, width).  Pair i of a section of n elements turns by theta ** (-2 i / n) radians per step of its axis; ``shared``: all axes
    share one ladder over the whole rotary part, pair p of it by theta ** (-2 p / sum(sections))."""
    sec = [int(s) for s in sections]
    if not sec or min(sec) < 2 or any(s % 2 for s in sec) or sum(sec) > 1024:
        raise ValueError(f"rotary_table: sections {sec} (even, at least 2 each, at most 1024 in all)")
    theta = float(theta)
    if not (theta > 0 and math.isfinite(theta)):
        raise ValueError("rotary_table: theta must be positive and finite")
    rotary, turns, axis = sum(sec), [], []
    for a, n in enumerate(sec):
        for i in range(n // 2):
            e = 2.0 * len(turns) / rotary if shared else 2.0 * i / n
            turns.append(theta ** -e / (2.0 * math.pi))
            axis.append(a)
    dev = torch.device(device)
    return RotaryTable(torch.tensor(turns, dtype=torch.float64).to(dev), torch.tensor(axis, dtype=torch.int32).to(dev), len(sec))


def rotary_axes(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, table: RotaryTable, *, heads: int, kv_heads: Optional[int] = None,
                d: int, pairing: str = "adjacent", out_q: Optional[torch.Tensor] = None, out_k: Optional[torch.Tensor] = None):
    """Turns ``q`` [tokens, heads * d] and ``k`` [tokens, kv_heads * d] (or ``None``) by their tokens' ``positions`` [tokens, axes] (int32 or
    fp32) in one launch; ``pairing``: "adjacent" turns elements 2 p and 2 p + 1 of a head, "halves" p and p + pairs.  A head's elements
    behind the rotary part pass through.  ``out_q`` / ``out_k`` may be ``q`` / ``k`` themselves.  Returns (q, k) turned (k ``None`` if not given)."""
    q = _matrix(q, "q")
    heads, d = int(heads), int(d)
    kv_heads = heads if kv_heads is None else int(kv_heads)
    if pairing not in ("adjacent", "halves"):
        raise ValueError(f"rotary_axes: pairing {pairing!r} (adjacent, halves)")
    n = q.shape[0]
    if heads < 1 or kv_heads < 1 or d < 1 or q.shape[1] != heads * d:
        raise ValueError(f"rotary_axes: q {tuple(q.shape)} for {heads} heads of {d}")
    if 2 * table.pairs > d:
        raise ValueError(f"rotary_axes: the table turns {2 * table.pairs} elements, a head has {d}")
    if k is not None:
        _matrix(k, "k", q.dtype, q.device)
        if k.shape != (n, kv_heads * d):
            raise ValueError(f"rotary_axes: k {tuple(k.shape)} for {n} tokens, {kv_heads} heads of {d}")
    elif out_k is not None:
        raise ValueError("rotary_axes: out_k without k")
    if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.float32):
        raise ValueError("rotary_axes: positions must be an int32 or fp32 tensor")
    _matrix(positions, "positions", positions.dtype, q.device)
    if positions.shape != (n, table.axes):
        raise ValueError(f"rotary_axes: positions {tuple(positions.shape)} for {n} tokens of {table.axes} axes")
    if table.device != q.device:
        raise ValueError(f"rotary_axes: table on {table.device}, tensors on {q.device}")
    outs = []
    for nm, t, o in (("q", q, out_q), ("k", k, out_k)):
        if t is None:
            outs.append(None)
            continue
        if o is None:
            o = torch.empty(t.shape, dtype=t.dtype, device=t.device)
        else:
            _matrix(o, f"out_{nm}", q.dtype, q.device)
            if o.shape != t.shape:
                raise ValueError(f"rotary_axes: out_{nm} {tuple(o.shape)}, {nm} {tuple(t.shape)}")
            _no_overlap(o, f"rotary_axes: out_{nm}", (("q", q), ("k", k), ("positions", positions)), (nm,))
        outs.append(o)
    oq, ok = outs
    if ok is not None and out_q is not None and out_k is not None:
        _no_overlap(oq, "rotary_axes: out_q", (("out_k", ok),))
    ds = RotaryDesc()
    ds.q, ds.out_q, ds.ldq, ds.ldoq = q.data_ptr(), oq.data_ptr(), _ld(q), _ld(oq)
    if k is not None:
        ds.k, ds.out_k, ds.ldk, ds.ldok = k.data_ptr(), ok.data_ptr(), _ld(k), _ld(ok)
    ds.positions, ds.ldp, ds.positions_f32 = positions.data_ptr(), _ld(positions), int(positions.dtype == torch.float32)
    ds.turns, ds.axis, ds.pairs, ds.axes = table.turns.data_ptr(), table.axis.data_ptr(), table.pairs, table.axes
    ds.tokens, ds.heads, ds.kv_heads, ds.d, ds.halves, ds.dtype = n, heads, kv_heads, d, int(pairing == "halves"), _DTYPES[q.dtype]
    with _device_of(q.device) as stream:
        table._use(stream)
        check(_lib.load().mv_rotary_axes(C.byref(ds), stream), "mv_rotary_axes")
    return oq, ok


# ---- gated residual norm ----------------------------------------------------------------------------------------------------------
Affine = Tuple[Optional[torch.Tensor], Optional[torch.Tensor], float]   # (gamma, beta, eps)


def _affine(t: Optional[torch.Tensor], name: str, c: int, like: torch.Tensor) -> Optional[int]:
    if t is None:
        return None
    if t.dtype != like.dtype or t.device != like.device or not t.is_contiguous() or t.numel() != c:
        raise ValueError(f"{name}: expected a contiguous {like.dtype} tensor of {c} elements on {like.device}")
    return t.data_ptr()


def gated_residual_norm(x: torch.Tensor, f: torch.Tensor, *, kind: str = "layer", alpha: float = 1.0, post: Optional[Affine] = None,
                        pre: Optional[Affine] = None, gate: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                        shift: Optional[torch.Tensor] = None, rows_per_group: Optional[int] = None, group_index: Optional[torch.Tensor] = None,
                        out: Optional[torch.Tensor] = None, norm_out: Optional[torch.Tensor] = None):
    """Ends one block and begins the next in one pass over the stream ``x`` and the block's output ``f`` (both [rows, C], C <= 16384):

        s = alpha * x + gate[g] * (N(f) * gamma + beta  with ``post = (gamma, beta, eps)``, else f)
        h = (N(s) * gamma + beta) * (1 + scale[g]) + shift[g]   with ``pre = (gamma, beta, eps)``; h reads s before its rounding

    N: ``kind`` "rms" or "layer"; a gamma or beta may be ``None``.  ``gate`` / ``scale`` / ``shift``: [groups, C] matrices, g the row's group --
    ``group_index`` (int32 per row: packed sequences) or row // ``rows_per_group``; with one group neither is needed.  A row whose
    group_index is no group is filled with NaN.  Returns (s, h), h ``None`` without ``pre``.  ``out`` may be ``x`` or ``f`` itself, ``norm_out`` too."""
    x = _matrix(x, "x")
    rows, c = x.shape
    _matrix(f, "f", x.dtype, x.device)
    if f.shape != x.shape:
        raise ValueError(f"gated_residual_norm: x {tuple(x.shape)}, f {tuple(f.shape)}")
    if kind not in ("rms", "layer"):
        raise ValueError(f"gated_residual_norm: kind {kind!r} (rms, layer)")
    if not 1 <= c <= 16384:
        raise ValueError(f"gated_residual_norm: {c} columns (1 .. 16384)")
    if pre is None and (scale is not None or shift is not None or norm_out is not None):
        raise ValueError("gated_residual_norm: scale / shift / norm_out belong to the norm in front of the next block (pre)")
    ds = GatedNormDesc()
    groups = None
    for nm, t in (("gate", gate), ("scale", scale), ("shift", shift)):
        if t is None:
            continue
        _matrix(t, nm, x.dtype, x.device)
        if t.shape[1] != c or t.shape[0] < 1 or (groups is not None and t.shape[0] != groups):
            raise ValueError(f"gated_residual_norm: {nm} {tuple(t.shape)} for {c} columns" + (f" and {groups} groups" if groups else ""))
        groups = t.shape[0]
    if rows_per_group is not None and group_index is not None:
        raise ValueError("gated_residual_norm: rows_per_group or group_index, not both")
    if group_index is not None:
        if groups is None:
            raise ValueError("gated_residual_norm: group_index without gate, scale or shift")
        if group_index.dtype != torch.int32 or group_index.shape != (rows,) or not group_index.is_contiguous() or group_index.device != x.device:
            raise ValueError(f"gated_residual_norm: group_index must be contiguous int32 [{rows}] on {x.device}")
        ds.group_index = group_index.data_ptr()
    elif rows_per_group is not None:
        rows_per_group = int(rows_per_group)
        if groups is None or rows_per_group < 1 or groups * rows_per_group < rows:
            raise ValueError(f"gated_residual_norm: {groups} groups of {rows_per_group} rows do not cover {rows}")
        ds.rows_per_group = min(rows_per_group, _I32_MAX)
    elif groups is not None and groups > 1:
        raise ValueError(f"gated_residual_norm: {groups} groups need rows_per_group or group_index")
    ins = (("x", x), ("f", f), ("gate", gate), ("scale", scale), ("shift", shift), ("group_index", group_index))
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        _matrix(out, "out", x.dtype, x.device)
        if out.shape != x.shape:
            raise ValueError(f"gated_residual_norm: out {tuple(out.shape)}, x {tuple(x.shape)}")
        _no_overlap(out, "gated_residual_norm: out", ins, ("x", "f"))
    if pre is not None:
        if norm_out is None:
            norm_out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        else:
            _matrix(norm_out, "norm_out", x.dtype, x.device)
            if norm_out.shape != x.shape:
                raise ValueError(f"gated_residual_norm: norm_out {tuple(norm_out.shape)}, x {tuple(x.shape)}")
            _no_overlap(norm_out, "gated_residual_norm: norm_out", ins, ("x", "f"))
        _no_overlap(norm_out, "gated_residual_norm: norm_out", (("out", out),))
        ds.pre_gamma, ds.pre_beta, ds.pre_eps = _affine(pre[0], "pre gamma", c, x), _affine(pre[1], "pre beta", c, x), float(pre[2])
        ds.norm_out, ds.ldh = norm_out.data_ptr(), _ld(norm_out)
    if post is not None:
        ds.post, ds.post_eps = 1, float(post[2])
        ds.post_gamma, ds.post_beta = _affine(post[0], "post gamma", c, x), _affine(post[1], "post beta", c, x)
    ds.x, ds.f, ds.stream_out = x.data_ptr(), f.data_ptr(), out.data_ptr()
    ds.ldx, ds.ldf, ds.lds = _ld(x), _ld(f), _ld(out)
    for nm, t, ld in (("gate", gate, "ldg"), ("scale", scale, "ldsc"), ("shift", shift, "ldsh")):
        if t is not None:
            setattr(ds, nm, t.data_ptr())
            setattr(ds, ld, _ld(t))
    ds.rows, ds.groups, ds.c = rows, groups or 1, c
    ds.layer, ds.dtype, ds.alpha = int(kind == "layer"), _DTYPES[x.dtype], float(alpha)
    with _device_of(x.device) as stream:
        check(_lib.load().mv_gated_residual_norm(C.byref(ds), stream), "mv_gated_residual_norm")
    return out, norm_out


# ---- int8 projection ------------------------------------------------------------------------------------------------------------------
class Int8Rows(_Held):
    """int8 rows with one scale each: row m stands for ``codes[m, :k] * scale[m]``.  ``codes`` is padded with zeros to a multiple of 128 columns."""

    def __init__(self, codes: torch.Tensor, scale: torch.Tensor, k: int):
        self.codes, self.scale, self.k, self.rows = codes, scale, k, codes.shape[0]
        self._hold(codes, scale)


def pack_weight_i8(codes: torch.Tensor, scale: torch.Tensor) -> Int8Rows:
    """:class:`Int8Rows` from int8 ``codes`` [N, K] and fp32 ``scale`` [N] (a checkpoint's weight: one scale per output channel), laid out for
    :func:`gemm_i8` once."""
    if codes.dim() != 2 or codes.dtype != torch.int8 or not _on_gpu(codes) or not 1 <= codes.shape[1] <= 131072:
        raise ValueError("pack_weight_i8: codes must be a CUDA int8 [N, K] tensor, K <= 131072")
    if scale.dtype != torch.float32 or scale.shape != (codes.shape[0],) or scale.device != codes.device:
        raise ValueError(f"pack_weight_i8: scale must be fp32 [{codes.shape[0]}] on {codes.device}")
    n, k = codes.shape
    packed = torch.zeros((n, -(-k // 128) * 128), dtype=torch.int8, device=codes.device)
    packed[:, :k] = codes
    return Int8Rows(packed, scale.clone(memory_format=torch.contiguous_format), k)


def quantize_rows_i8(x: torch.Tensor) -> Int8Rows:
    """Each row of ``x`` [M, K] (fp16 | bf16) as int8 codes and one scale: scale = max|x| / 127, code = 127 x / max|x| rounded to nearest, ties
    to even.  A row of zeros has scale 0; a row that holds an infinity or NaN keeps that as its scale (its products are NaN)."""
    x = _matrix(x, "x")
    m, k = x.shape
    if not 1 <= k <= 131072:
        raise ValueError(f"quantize_rows_i8: {k} columns (1 .. 131072)")
    codes = torch.empty((m, -(-k // 128) * 128), dtype=torch.int8, device=x.device)
    scale = torch.empty((m,), dtype=torch.float32, device=x.device)
    with _device_of(x.device) as stream:
        check(_lib.load().mv_quantize_rows_i8(x.data_ptr(), _ld(x), m, k, _DTYPES[x.dtype], codes.data_ptr(), codes.shape[1], scale.data_ptr(), stream),
              "mv_quantize_rows_i8")
    return Int8Rows(codes, scale, k)


def _i8_checks(what: str, m: int, w: Int8Rows, device, dtype, bias, residual, act, out):
    if dtype not in _DTYPES:
        raise ValueError(f"{what}: dtype {dtype} (fp16, bf16)")
    if act not in (MV_ACT_NONE, MV_ACT_SILU):
        raise ValueError(f"{what}: activation {act}")
    if w.device != device:
        raise ValueError(f"{what}: weight on {w.device}, rows on {device}")
    n = w.rows
    if n < 1:
        raise ValueError(f"{what}: a weight without rows")
    ds = GemmI8Desc()
    if bias is not None:
        if bias.dtype != dtype or bias.device != device or not bias.is_contiguous() or bias.numel() != n:
            raise ValueError(f"{what}: bias must be a contiguous {dtype} tensor of {n} elements on {device}")
        ds.bias = bias.data_ptr()
    if residual is not None:
        _matrix(residual, "residual", dtype, device)
        if residual.shape != (m, n):
            raise ValueError(f"{what}: residual {tuple(residual.shape)}, the product is {(m, n)}")
        ds.residual, ds.ldr = residual.data_ptr(), _ld(residual)
    if out is not None:
        _matrix(out, "out", dtype, device)
        if out.shape != (m, n):
            raise ValueError(f"{what}: out {tuple(out.shape)}, the product is {(m, n)}")
        _no_overlap(out, f"{what}: out", (("residual", residual), ("bias", bias)), ("residual",))
    ds.M, ds.N, ds.kp, ds.ldw = m, n, w.codes.shape[1], w.codes.shape[1]
    ds.w, ds.w_scale, ds.act, ds.dtype = w.codes.data_ptr(), w.scale.data_ptr(), int(act), _DTYPES[dtype]
    return ds


def gemm_i8(a: Int8Rows, w: Int8Rows, *, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None, act: int = MV_ACT_NONE,
            dtype: torch.dtype = torch.float16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(a_scale[m] * w_scale[n] * sum_k a[m, k] w[n, k] + bias) + residual as ``dtype`` [M, N]; the sum of products is exact (int32).
    ``out`` may be ``residual`` itself."""
    if a.k != w.k:
        raise ValueError(f"gemm_i8: rows of {a.k}, weight of {w.k}")
    ds = _i8_checks("gemm_i8", a.rows, w, a.device, dtype, bias, residual, act, out)
    if out is None:
        out = torch.empty((a.rows, w.rows), dtype=dtype, device=a.device)
    ds.a, ds.a_scale, ds.lda, ds.out, ds.ldo = a.codes.data_ptr(), a.scale.data_ptr(), a.codes.shape[1], out.data_ptr(), _ld(out)
    with _device_of(a.device) as stream:
        a._use(stream)
        w._use(stream)
        check(_lib.load().mv_gemm_i8(C.byref(ds), stream), "mv_gemm_i8")
    return out


def linear_i8(x: torch.Tensor, w: Int8Rows, *, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None, act: int = MV_ACT_NONE,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`gemm_i8` of :func:`quantize_rows_i8` (``x``): a projection whose weight and activations are multiplied in 8 bits."""
    x = _matrix(x, "x")
    if x.shape[1] != w.k:
        raise ValueError(f"linear_i8: x {tuple(x.shape)}, weight of {w.k}")
    if out is not None and isinstance(out, torch.Tensor) and out.dim() == 2:
        _no_overlap(out, "linear_i8: out", (("x", x),))
    return gemm_i8(quantize_rows_i8(x), w, bias=bias, residual=residual, act=act, dtype=x.dtype, out=out)
