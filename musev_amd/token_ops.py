"""Token-transformer operators over the C ABI of include/musev_tokens.h: packed attention, rotary positions with several axes, the gated
residual norm and the int8 projection.  They are part of :mod:`musev_amd.ops` (``from musev_amd import ops; ops.attention_packed(...)``)
and follow its manner: 2-D row matrices with unit inner stride, no CPU path, launches on the current stream of the tensors' device.
fp16 and bf16; forward only, like the rest of the framework: a tensor that requires gradients is refused while gradients are recorded, and
so is one that carries a forward-mode tangent.

Each call reads its tensors on the stream it is made on: a tensor made on another stream has to be finished there first.  Nothing is kept
between calls; what a call needs besides its arguments is allocated for that call (inside a graph capture: from the capture's pool), so
concurrent calls and several captured graphs never share it.  A graph refers to the plan, table or codes it was captured with: keep them.
"""
from __future__ import annotations

import collections
import ctypes as C
import heapq
import itertools
import math
import operator
import struct
from typing import Callable, List, Optional, Sequence, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import MV_ACT_NONE, MV_ACT_SILU, AttnPackedDesc, GatedNormDesc, GemmI8Desc, LinearI8Desc, RotaryDesc, check

__all__ = ["AttentionPlan", "attention_plan", "attention_packed", "RotaryTable", "rotary_table", "rotary_axes", "gated_residual_norm",
           "Int8Rows", "pack_weight_i8", "quantize_rows_i8", "gemm_i8", "linear_i8"]

_DTYPES = {torch.float16: 0, torch.bfloat16: 1}
_I32_MAX = 2 ** 31 - 1
_F32_MAX = 2.0 ** 128 - 2.0 ** 104

# A small call's time is the host's: checks read each tensor's geometry once, a descriptor is packed in one go, the stream is asked for as a
# raw handle (a torch built without a GPU has none: the rest of the package is imported beside it all the same).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", None)


def _packer(desc) -> Callable[..., bytes]:
    """packs a descriptor's fields, in their order, into the bytes of the C struct (0 for a null pointer)"""
    code = {C.c_void_p: "P", C.c_int64: "q", C.c_int32: "i", C.c_float: "f"}
    form = struct.Struct("@" + "".join(code[t] for _, t in desc._fields_) + "0P")
    assert form.size == C.sizeof(desc)
    return form.pack


_pack_attention, _pack_rotary, _pack_norm, _pack_gemm, _pack_linear = (_packer(d) for d in (AttnPackedDesc, RotaryDesc, GatedNormDesc, GemmI8Desc,
                                                                                           LinearI8Desc))


def _on_gpu(t: torch.Tensor) -> bool:
    return t.is_cuda


def _launch(entry: str, desc: bytes, dev: int, held: Sequence["_Held"] = ()) -> None:
    """one call of the C ABI on device ``dev``'s current stream"""
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return _launch(entry, desc, dev, held)
    stream = _raw_stream(dev)
    for h in held:
        if stream not in h._streams:
            h._use(stream)
    status = getattr(_lib._lib or _lib.load(), entry)(desc, stream)
    if status:
        check(status, entry)


def _no_gradients(name: str, t: torch.Tensor) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: requires gradients, and this operator has none to give: call it under torch.no_grad() or detach the tensor")
    if t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name}: carries a forward-mode tangent, and this operator has no derivative to give: unpack the tensor first")


def _matrix(t: torch.Tensor, name: str, dtype: Optional[torch.dtype] = None, dev: Optional[int] = None) -> Tuple[int, int, int]:
    """(rows, columns, row stride) of a 2-D tensor with unit inner stride on the GPU; a single row has no stride of its own: its width stands in"""
    if not isinstance(t, torch.Tensor) or t.ndim != 2:
        raise ValueError(f"{name}: expected a 2-D tensor, got {tuple(t.shape) if isinstance(t, torch.Tensor) else type(t).__name__}")
    rows, cols = t.shape
    ld, inner = t.stride()
    if inner != 1 and cols > 1:
        raise ValueError(f"{name}: expected unit inner stride, got shape {(rows, cols)} strides {(ld, inner)}")
    if dev is None and not _on_gpu(t) or (t.dtype not in _DTYPES if dtype is None else t.dtype != dtype):
        raise ValueError(f"{name}: expected a CUDA {'fp16 | bf16' if dtype is None else dtype} tensor, got {t.dtype} on {t.device}")
    if dev is not None and t.get_device() != dev:
        raise ValueError(f"{name}: on {t.device}, the other tensors are on device {dev}")
    if t.requires_grad or forward_ad._current_level >= 0:   # (a level is open: tensors may carry tangents)
        _no_gradients(name, t)
    if rows <= 1:
        return rows, cols, cols
    if ld < cols or ld > _I32_MAX:
        raise ValueError(f"{name}: row stride {ld} for {cols} columns")
    return rows, cols, ld


def _ld(t: torch.Tensor) -> int:
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

    def _hold(self, *tensors: torch.Tensor, ready: Optional[torch.cuda.Event] = None) -> None:
        self._tensors, self._ready = tensors, ready
        self.device = tensors[0].device
        self._dev = tensors[0].get_device()
        self._streams = {_raw_stream(self._dev)} if tensors[0].is_cuda else set()

    def _made_of(self) -> tuple:
        """the constructor's arguments: a copy (copy.deepcopy, pickle) is made anew, with the addresses of its own memory"""
        raise NotImplementedError

    def __reduce__(self):
        if self._ready is not None and not torch.cuda.is_current_stream_capturing():   # (whoever copies the memory reads it on the current stream)
            torch.cuda.current_stream(self.device).wait_event(self._ready)
        return type(self), self._made_of()

    def _use(self, stream: int) -> None:
        # (first use on a stream) what was filled without a wait for it is waited for there, and the allocator may not hand the memory out again while
        # a launch there still reads it
        if not torch.cuda.is_current_stream_capturing():
            here = torch.cuda.current_stream(self.device)
            if self._ready is not None:
                here.wait_event(self._ready)
            for t in self._tensors:
                t.record_stream(here)
            self._streams.add(stream)


# ---- packed attention ---------------------------------------------------------------------------------------------------------
class AttentionPlan(_Held):
    """the work list of :func:`attention_packed` for one set of sequence lengths (:func:`attention_plan`)"""

    def __init__(self, q_lens, kv_lens, heads, kv_heads, d, causal, scale, items, joins, join_rows, ws_rows, kv_first=None, ready=None):
        kv_first = _behind(kv_lens) if kv_first is None else kv_first
        self.q_lens, self.kv_lens, self.kv_first = tuple(q_lens), tuple(kv_lens), tuple(kv_first)
        self.heads, self.kv_heads, self.d, self.causal, self.scale = heads, kv_heads, d, causal, scale
        self.total_q, self.total_kv = sum(q_lens), max((f + n for f, n in zip(kv_first, kv_lens) if n), default=0)   # (rows of q; of k and v)
        self.n_items, self.n_joins, self.join_rows, self.ws_rows = items.shape[0], joins.shape[0], join_rows, ws_rows
        self._hold(items, joins, ready=ready)
        self._tables = items.data_ptr(), joins.data_ptr()
        self._workspace = 4 * ws_rows * kv_heads * (d + 2)   # mv_attention_packed_workspace_bytes

    def _made_of(self) -> tuple:
        return (self.q_lens, self.kv_lens, self.heads, self.kv_heads, self.d, self.causal, self.scale, *self._tensors, self.join_rows, self.ws_rows, self.kv_first)


def _integers(v, name: str) -> List[int]:
    if isinstance(v, torch.Tensor):
        if v.is_cuda:
            raise ValueError(f"{name}: lengths are host integers (reading them from the GPU would wait for it)")
        v = v.tolist()
    return [operator.index(x) for x in v]


def _lens(v, name: str) -> List[int]:
    v = _integers(v, name)
    if not v or min(v) < 0 or sum(v) > _I32_MAX:
        raise ValueError(f"{name}: expected at least one length, none negative, at most 2^31 - 1 rows in all")
    return v


def _behind(lens: Sequence[int]) -> List[int]:
    """first rows of sequences that stand one behind the other"""
    return [0, *itertools.accumulate(lens[:-1])]


TILE_ROWS = 128   # packed rows per item
# The least keys of a part: an item's parts each write and the join reads back (d + 2) fp32 per row.
MIN_PART = 128
BLOCKS = 512      # two blocks on each of the 256 CUs
LATE_PART = 1024  # keys of a part of a block that would run late


def _plan_items(ql: Sequence[int], kl: Sequence[int], group: int, kv_heads: int, causal: bool, d: int = 128, first: Optional[Sequence[int]] = None):
    """(items, joins, workspace rows): see include/musev_tokens.h.  An item's keys end with what its last query sees.  Where the items alone would
    leave CUs idle, or one item would outlast the others, its keys are split into parts of 1 / BLOCKS of all the work or more (`_cheapest_parts`;
    `_late_parts`: or where a last round would hold few of them); the longest items come first."""
    tiles, q_row = [], 0
    for q, kv, k_row in zip(ql, kl, _behind(kl) if first is None else first):
        for m0 in range(0, q * group, TILE_ROWS):
            last = min(m0 + TILE_ROWS, q * group) - 1
            tiles.append((q_row, q, k_row, kv, m0, max(0, min(kv, last // group + kv - q + 1)) if causal else kv))
        q_row += q
    items, joins, ws = [], [], 0
    part = max(MIN_PART, -(-sum(t[5] for t in tiles) * kv_heads // BLOCKS))
    part = -(-part // 64) * 64
    parts = [max(1, (t[5] + part // 2) // part) for t in tiles]
    if max(parts, default=1) > 1:
        parts = _cheapest_parts([(min(TILE_ROWS, t[1] * group - t[4]), t[5]) for t in tiles], part, kv_heads, d)
    if max(parts, default=1) == 1 and BLOCKS < len(tiles) * kv_heads <= 8 * BLOCKS:
        parts = _late_parts([t[5] for t in tiles], kv_heads)
    for (q_row, q, k_row, kv, m0, end), n in zip(tiles, parts):
        if n == 1:
            items.append((q_row, q, k_row, kv, m0, 0, end, -1))
            continue
        size = -(-(-(-end // n)) // 64) * 64
        n = -(-end // size)
        rows = min(TILE_ROWS, q * group - m0)
        for s in range(n):
            items.append((q_row, q, k_row, kv, m0, s * size, min(end, (s + 1) * size), ws + s * rows))
        joins.append((q_row, q, kv, m0, ws, n, rows, 0))
        ws += n * rows
    items.sort(key=lambda i: i[5] - i[6])
    return items, joins, ws


def _cheapest_parts(tiles: Sequence[Tuple[int, int]], part: int, kv_heads: int, d: int) -> List[int]:
    """Parts of every tile (its rows, its keys), of ``part`` keys or a multiple of that, whichever costs least: the longest part's tiles of 64 keys
    1.22 us each (at head dim 128), the join 2.7 us and 0.64 us for each MB of sums that parts hand over -- fitted to 24 sets of lengths at five sizes
    of parts, within 10 %.  Measured (us, parts of 1 / BLOCKS / cheapest): 587 tokens of 32 / 4 heads x 104 24.2 / 16.7; 3 x 700 of 8 / 2 x 64 20.0 / 14.8;
    4 x 300 of 8 x 64 12.9 / 9.7; 128 tokens over 8192 keys of 8 x 128 24.8 / 22.9; 1500 of 4 / 1 x 128 23.1 / 20.1; one token per request: the same."""
    counts = collections.Counter(tiles)
    per_tile = 1.22 * (0.35 + 0.65 * -(-d // 16) / 8)
    least = sum(end * n for (_, end), n in counts.items()) * kv_heads // BLOCKS   # (keys of a block if all were busy to the end)
    best, choice = math.inf, part
    for f in (1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 8.0, math.inf):
        size, longest, shared = f * part, least, 0
        for (rows, end), n in counts.items():
            k = max(1, int(end / size + 0.5))
            longest = max(longest, -(-end // k))
            if k > 1:
                shared += rows * k * n
        cost = per_tile * -(-longest // 64) + (2.7 + 0.64e-6 * 4 * shared * kv_heads * (d + 2) if shared else 0.0)
        if cost < 0.97 * best:
            best, choice = cost, size
    return [max(1, int(end / choice + 0.5)) for _, end in tiles]


def _late_parts(ends: Sequence[int], kv_heads: int) -> List[int]:
    """Parts of every tile (`ends`: its keys) where there are a few rounds of blocks: blocks that would outlast the mean are split to end with the
    others, where they are few and long enough to pay for the join of their parts.  Measured (us, whole / split, late blocks x their keys): 12 heads
    over 6000 keys 272 / 227 [60 x 6000], 6 over 13 312 590 / 514 [114], 8 over 13 312 573 / 516 [320]; but 8 over 4 x 3000 149 / 162 [256 x 3000], 8 over
    3 x 4500 262 / 272 [352 x 4500], 8 over 6 x 1500 46.6 / 47.0 [64 x 1500]."""
    parts = [1] * len(ends)
    if max(ends) < 2 * LATE_PART:
        return parts
    order = sorted(range(len(ends)), key=lambda i: -ends[i])
    mean = sum(ends) * kv_heads // BLOCKS

    def rooms(split):
        """(tile, keys that fit in before the mean where its last block starts) in order; tiles for which ``split`` holds are cut to that size"""
        busy = [0] * BLOCKS
        for i in order:
            start = busy[0]
            if split(i):
                start = heapq.nsmallest(kv_heads, busy)[-1]
                parts[i] = -(-ends[i] // max(LATE_PART, mean - start))
            for _ in range(kv_heads * parts[i]):
                start = busy[0]
                heapq.heapreplace(busy, start + ends[i] // parts[i])
            yield i, mean - start

    late = {i for i, room in rooms(lambda i: False) if ends[i] > room + LATE_PART}
    late = {i for i in late if ends[i] >= 32 * kv_heads * len(late)}
    if late:
        for _ in rooms(lambda i: i in late):
            pass
    return parts


def attention_plan(q_lens: Sequence[int], kv_lens: Optional[Sequence[int]] = None, *, heads: int, kv_heads: Optional[int] = None, d: int,
                   causal: bool = True, scale: Optional[float] = None, kv_first: Optional[Sequence[int]] = None,
                   device: Union[str, torch.device] = "cuda") -> AttentionPlan:
    """The plan of :func:`attention_packed` over ``len(q_lens)`` sequences of ``q_lens[i]`` query and ``kv_lens[i]`` key rows (default: as
    many), host integers, zero allowed.  ``causal``: query i of a sequence sees keys j <= i + kv_len - q_len -- the new tokens stand at the
    end of their keys.  ``scale``: of the scores, default d ** -0.5.  ``kv_first``: the row of ``k`` / ``v`` at which each sequence's keys begin, default one
    sequence behind the other; with it a cache keeps room behind every sequence, and sequences may share rows.  Made once per set of lengths and
    used for every layer (lengths that grow need a plan per step: 100 us of host time for 16
    requests of one token over 86 000 keys, 200 for 128, beside the GPU's work).
    The list is uploaded on the current stream without a wait for the work queued there; other streams wait for it at the plan's first use.
    A graph holds the plan that it was captured with: its replays come behind the upload (torch.cuda.graph waits for it), and no plan is
    made while a graph is captured."""
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
    if kv_first is None:
        first = _behind(kl)
    else:
        first = _integers(kv_first, "kv_first")
        if len(first) != len(kl) or min(first) < 0 or max(f + n for f, n in zip(first, kl)) > _I32_MAX:
            raise ValueError("attention_plan: kv_first: expected a row for each sequence, none negative, keys within 2^31 - 1 rows")
    if max(ql) * (heads // kv_heads) > _I32_MAX:
        raise ValueError("attention_plan: more than 2^31 - 1 (query, head) rows per key / value head")
    scale = d ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= 1e6:
        raise ValueError(f"attention_plan: scale {scale} (at most 1e6 in size)")
    dev = torch.device(device)
    if dev.type == "cuda":
        if torch.cuda.is_current_stream_capturing():
            raise ValueError("attention_plan: a plan's list comes from the host and cannot be part of a graph: make it before the capture")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
    items, joins, ws_rows = _plan_items(ql, kl, heads // kv_heads, kv_heads, bool(causal), d, first)
    # One upload, from pinned memory: from pageable memory the host would wait for all work queued on the stream.  (The allocator keeps the pinned
    # block until the copy is done.)
    table, ready = torch.tensor((items + joins) or [(0,) * 8], dtype=torch.int32, device="cpu", pin_memory=dev.type == "cuda"), None
    table = table.to(dev, non_blocking=True)
    if dev.type == "cuda":
        ready = torch.cuda.Event()
        ready.record(torch.cuda.current_stream(dev))
    n = len(items)
    return AttentionPlan(ql, kl, heads, kv_heads, d, bool(causal), scale, table[:n], table[n:n + len(joins)], max((j[6] for j in joins), default=0), ws_rows,
                         first, ready)


def attention_packed(plan: AttentionPlan, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Softmax attention of packed sequences: ``q`` [>= total_q, heads * d], ``k`` / ``v`` [>= total_kv, kv_heads * d], fp16 or bf16, any row
    stride that keeps rows 16-byte aligned (column slices of a fused projection).  Returns [total_q, heads * d], or writes the first
    total_q rows of ``out`` and leaves the rows behind them as they were.  A query that sees no key gives 0; what a query does not see --
    later tokens, other sequences, rows behind the last one -- does not reach its output, NaN and infinities included."""
    rows, cols, ldq = _matrix(q, "q")
    dtype, dev = q.dtype, q.get_device()
    hd, kvd = plan.heads * plan.d, plan.kv_heads * plan.d
    if cols != hd or rows < plan.total_q:
        raise ValueError(f"attention_packed: q {(rows, cols)}, the plan has {plan.total_q} rows of {hd}")
    rows, cols, ldk = _matrix(k, "k", dtype, dev)
    if cols != kvd or rows < plan.total_kv:
        raise ValueError(f"attention_packed: k {(rows, cols)}, the plan has {plan.total_kv} rows of {kvd}")
    rows, cols, ldv = _matrix(v, "v", dtype, dev)
    if cols != kvd or rows < plan.total_kv:
        raise ValueError(f"attention_packed: v {(rows, cols)}, the plan has {plan.total_kv} rows of {kvd}")
    if plan._dev != dev:
        raise ValueError(f"attention_packed: plan on {plan.device}, tensors on {q.device}")
    if out is None:
        out, ldo = q.new_empty((plan.total_q, hd)), hd
    else:
        rows, cols, ldo = _matrix(out, "out", dtype, dev)
        if cols != hd or rows < plan.total_q:
            raise ValueError(f"attention_packed: out {(rows, cols)}, the plan has {plan.total_q} rows of {hd}")
        _no_overlap(out[:plan.total_q], "attention_packed: out", (("q", q), ("k", k), ("v", v)))
    pq, pk, pv, po = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    if (pq | pk | pv | po) & 15 or (ldq | ldk | ldv | ldo) & 7 or max(ldk, ldv) > 1 << 23:
        raise ValueError(f"attention_packed: rows must be 16-byte aligned and k / v rows at most 2^23 elements apart, row strides {(ldq, ldk, ldv, ldo)}")
    ws = torch.empty(plan._workspace, dtype=torch.uint8, device=q.device) if plan._workspace else None
    items, joins = plan._tables
    _launch("mv_attention_packed", _pack_attention(pq, pk or pq, pv or pq, po, items, joins, ws.data_ptr() if ws is not None else 0,   # (no key: not read)
                                                   plan._workspace, plan.ws_rows, plan.n_items, plan.n_joins, plan.join_rows, ldq, ldk, ldv, ldo,
                                                   plan.heads, plan.kv_heads, plan.d, _DTYPES[dtype], plan.causal, plan.scale), dev, (plan,))
    return out


# ---- rotary positions ----------------------------------------------------------------------------------------------------------
class RotaryTable(_Held):
    """axis and turns per position step of every pair of a head (:func:`rotary_table`)"""

    def __init__(self, turns: torch.Tensor, axis: torch.Tensor, axes: int):
        self.pairs, self.axes = turns.numel(), axes
        self._hold(turns, axis)
        self._turns, self._axis = turns.data_ptr(), axis.data_ptr()

    def _made_of(self) -> tuple:
        return (*self._tensors, self.axes)


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
    return RotaryTable(torch.tensor(turns, dtype=torch.float64, device="cpu").to(dev), torch.tensor(axis, dtype=torch.int32, device="cpu").to(dev), len(sec))


def rotary_axes(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, table: RotaryTable, *, heads: int, kv_heads: Optional[int] = None,
                d: int, pairing: str = "adjacent", out_q: Optional[torch.Tensor] = None, out_k: Optional[torch.Tensor] = None):
    """Turns ``q`` [tokens, heads * d] and ``k`` [tokens, kv_heads * d] (or ``None``) by their tokens' ``positions`` [tokens, axes] (int32 or
    fp32) in one launch; ``pairing``: "adjacent" turns elements 2 p and 2 p + 1 of a head, "halves" p and p + pairs.  A head's elements
    behind the rotary part pass through.  ``out_q`` / ``out_k`` may be ``q`` / ``k`` themselves.  Returns (q, k) turned (k ``None`` if not given)."""
    n, cols, ldq = _matrix(q, "q")
    dtype, dev = q.dtype, q.get_device()
    kv_heads = heads if kv_heads is None else kv_heads
    if pairing not in ("adjacent", "halves"):
        raise ValueError(f"rotary_axes: pairing {pairing!r} (adjacent, halves)")
    if heads < 1 or kv_heads < 1 or d < 1 or cols != heads * d:
        raise ValueError(f"rotary_axes: q {(n, cols)} for {heads} heads of {d}")
    if 2 * table.pairs > d:
        raise ValueError(f"rotary_axes: the table turns {2 * table.pairs} elements, a head has {d}")
    pk = pok = ldk = ldok = 0
    if k is not None:
        rows, cols, ldk = _matrix(k, "k", dtype, dev)
        if rows != n or cols != kv_heads * d:
            raise ValueError(f"rotary_axes: k {(rows, cols)} for {n} tokens, {kv_heads} heads of {d}")
        pk = k.data_ptr()
    elif out_k is not None:
        raise ValueError("rotary_axes: out_k without k")
    if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.float32):
        raise ValueError("rotary_axes: positions must be an int32 or fp32 tensor")
    rows, cols, ldp = _matrix(positions, "positions", positions.dtype, dev)
    if rows != n or cols != table.axes:
        raise ValueError(f"rotary_axes: positions {(rows, cols)} for {n} tokens of {table.axes} axes")
    if table._dev != dev:
        raise ValueError(f"rotary_axes: table on {table.device}, tensors on {q.device}")
    if out_q is None:
        oq, ldoq = torch.empty_like(q), heads * d   # (a matrix with gaps between its rows gets one without)
    else:
        oq, ldoq = out_q, _rotary_out("q", q, out_q, (("q", q), ("k", k), ("positions", positions)), dtype, dev)
    ok = None
    if k is not None:
        if out_k is None:
            ok, ldok = torch.empty_like(k), kv_heads * d
        else:
            ok, ldok = out_k, _rotary_out("k", k, out_k, (("q", q), ("k", k), ("positions", positions)), dtype, dev)
            if out_q is not None:
                _no_overlap(oq, "rotary_axes: out_q", (("out_k", ok),))
        pok = ok.data_ptr()
    _launch("mv_rotary_axes", _pack_rotary(q.data_ptr(), pk, oq.data_ptr(), pok, positions.data_ptr(), table._turns, table._axis, n, ldq, ldk, ldoq, ldok,
                                           ldp, heads, kv_heads, d, table.pairs, table.axes, pairing == "halves", positions.dtype == torch.float32,
                                           _DTYPES[dtype]), dev, (table,))
    return oq, ok


def _rotary_out(nm: str, t: torch.Tensor, o: torch.Tensor, ins, dtype: torch.dtype, dev: int) -> int:
    _, _, ld = _matrix(o, f"out_{nm}", dtype, dev)
    if o.shape != t.shape:
        raise ValueError(f"rotary_axes: out_{nm} {tuple(o.shape)}, {nm} {tuple(t.shape)}")
    _no_overlap(o, f"rotary_axes: out_{nm}", ins, (nm,))
    return ld


# ---- gated residual norm ----------------------------------------------------------------------------------------------------------
Affine = Tuple[Optional[torch.Tensor], Optional[torch.Tensor], float]   # (gamma, beta, eps)


def _affine(t: Optional[torch.Tensor], name: str, c: int, dtype: torch.dtype, dev: int) -> int:
    if t is None:
        return 0
    if t.dtype != dtype or t.get_device() != dev or not t.is_contiguous() or t.numel() != c:
        raise ValueError(f"{name}: expected a contiguous {dtype} tensor of {c} elements on device {dev}")
    if t.requires_grad or forward_ad._current_level >= 0:
        _no_gradients(name, t)
    return t.data_ptr()


def gated_residual_norm(x: torch.Tensor, f: torch.Tensor, *, kind: str = "layer", alpha: float = 1.0, post: Optional[Affine] = None,
                        pre: Optional[Affine] = None, gate: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                        shift: Optional[torch.Tensor] = None, rows_per_group: Optional[int] = None, group_index: Optional[torch.Tensor] = None,
                        out: Optional[torch.Tensor] = None, norm_out: Optional[torch.Tensor] = None):
    """Ends one block and begins the next in one pass over the stream ``x`` and the block's output ``f`` (both [rows, C], C <= 16384):

        s = alpha * x + gate[g] * (N(f) * gamma + beta  with ``post = (gamma, beta, eps)``, else f)
        h = (N(s) * gamma + beta) * (1 + scale[g]) + shift[g]   with ``pre = (gamma, beta, eps)``; h reads s before its rounding

    N: ``kind`` "rms" or "layer"; a gamma or beta may be ``None``.  ``gate`` / ``scale`` / ``shift``: [groups, C] matrices, g the row's group --
    ``group_index`` (int32 per row: packed sequences) or row // ``rows_per_group``; with one group neither is needed.  Statistics are
    fp32: values up to about 1e16 in size.  A row whose group_index is no group is filled with NaN.  Returns (s, h), h ``None`` without
    ``pre``.  ``out`` may be ``x`` or ``f`` itself, ``norm_out`` too."""
    rows, c, ldx = _matrix(x, "x")
    dtype, dev = x.dtype, x.get_device()
    frows, fc, ldf = _matrix(f, "f", dtype, dev)
    if frows != rows or fc != c:
        raise ValueError(f"gated_residual_norm: x {(rows, c)}, f {(frows, fc)}")
    if kind not in ("rms", "layer"):
        raise ValueError(f"gated_residual_norm: kind {kind!r} (rms, layer)")
    if not 1 <= c <= 16384:
        raise ValueError(f"gated_residual_norm: {c} columns (1 .. 16384)")
    if pre is None and (scale is not None or shift is not None or norm_out is not None):
        raise ValueError("gated_residual_norm: scale / shift / norm_out belong to the norm in front of the next block (pre)")
    groups, mods = 0, []
    for nm, t in (("gate", gate), ("scale", scale), ("shift", shift)):
        if t is None:
            mods.append((0, 0))
            continue
        grows, gc, ld = _matrix(t, nm, dtype, dev)
        if gc != c or grows < 1 or (groups and grows != groups):
            raise ValueError(f"gated_residual_norm: {nm} {(grows, gc)} for {c} columns" + (f" and {groups} groups" if groups else ""))
        groups = grows
        mods.append((t.data_ptr(), ld))
    index = per = 0
    if group_index is not None:
        if rows_per_group is not None:
            raise ValueError("gated_residual_norm: rows_per_group or group_index, not both")
        if not groups:
            raise ValueError("gated_residual_norm: group_index without gate, scale or shift")
        if group_index.dtype != torch.int32 or group_index.shape != (rows,) or not group_index.is_contiguous() or group_index.get_device() != dev:
            raise ValueError(f"gated_residual_norm: group_index must be contiguous int32 [{rows}] on {x.device}")
        index = group_index.data_ptr()
    elif rows_per_group is not None:
        per = int(rows_per_group)
        if not groups or per < 1 or groups * per < rows:
            raise ValueError(f"gated_residual_norm: {groups} groups of {per} rows do not cover {rows}")
        per = min(per, _I32_MAX)
    elif groups > 1:
        raise ValueError(f"gated_residual_norm: {groups} groups need rows_per_group or group_index")
    for nm, a in (("post", post), ("pre", pre)):
        if a is not None and not 0.0 <= a[2] <= _F32_MAX:
            raise ValueError(f"gated_residual_norm: {nm} eps {a[2]} (a finite fp32 number, not negative)")
    if abs(alpha) > _F32_MAX and not math.isinf(alpha):
        raise ValueError(f"gated_residual_norm: alpha {alpha} is past fp32")
    given = out is not None or norm_out is not None
    if out is None:
        out, lds = torch.empty_like(x), c
    else:
        lds = _matrix(out, "out", dtype, dev)[2]
        if out.shape != x.shape:
            raise ValueError(f"gated_residual_norm: out {tuple(out.shape)}, x {(rows, c)}")
    pre_gamma = pre_beta = ldh = ph = 0
    pre_eps = 0.0
    if pre is not None:
        pre_gamma, pre_beta, pre_eps = _affine(pre[0], "pre gamma", c, dtype, dev), _affine(pre[1], "pre beta", c, dtype, dev), pre[2]
        if norm_out is None:
            norm_out, ldh = torch.empty_like(x), c
        else:
            ldh = _matrix(norm_out, "norm_out", dtype, dev)[2]
            if norm_out.shape != x.shape:
                raise ValueError(f"gated_residual_norm: norm_out {tuple(norm_out.shape)}, x {(rows, c)}")
        ph = norm_out.data_ptr()
    post_gamma = post_beta = 0
    post_eps = 0.0
    if post is not None:
        post_gamma, post_beta, post_eps = _affine(post[0], "post gamma", c, dtype, dev), _affine(post[1], "post beta", c, dtype, dev), post[2]
    if given:
        ins = (("x", x), ("f", f), ("gate", gate), ("scale", scale), ("shift", shift), ("group_index", group_index)) + tuple(
            (nm, t) for nm, a in (("post", post), ("pre", pre)) if a is not None for t in a[:2])
        _no_overlap(out, "gated_residual_norm: out", ins, ("x", "f"))
        if norm_out is not None:
            _no_overlap(norm_out, "gated_residual_norm: norm_out", ins, ("x", "f"))
            _no_overlap(norm_out, "gated_residual_norm: norm_out", (("out", out),))
    (pg, ldg), (psc, ldsc), (psh, ldsh) = mods
    _launch("mv_gated_residual_norm", _pack_norm(x.data_ptr(), f.data_ptr(), out.data_ptr(), ph, post_gamma, post_beta, pre_gamma, pre_beta, pg, psc, psh,
                                                 index, rows, groups or 1, per, c, ldx, ldf, lds, ldh, ldg, ldsc, ldsh, post is not None, kind == "layer",
                                                 _DTYPES[dtype], alpha, post_eps, pre_eps), dev)
    return out, norm_out


# ---- int8 projection ------------------------------------------------------------------------------------------------------------------
_I8_MAX_K = 131071   # K * 128 * 128 < 2^31: the sum of any int8 products fits 32 bits


class Int8Rows(_Held):
    """int8 rows with one scale each: row m stands for ``codes[m, :k] * scale[m]``.  ``codes`` is padded with zeros to a multiple of 128 columns."""

    def __init__(self, codes: torch.Tensor, scale: torch.Tensor, k: int):
        if not 1 <= k <= _I8_MAX_K or codes.dtype != torch.int8 or codes.ndim != 2 or not codes.is_contiguous() or codes.shape[1] != -(-k // 128) * 128 or \
                scale.dtype != torch.float32 or scale.shape != codes.shape[:1] or not scale.is_contiguous() or scale.device != codes.device:
            raise ValueError(f"Int8Rows: codes must be contiguous int8 [rows, {k} rounded up to 128] and scale contiguous fp32 [rows] beside them")
        self.codes, self.scale, self.k, self.rows, self.kp = codes, scale, k, codes.shape[0], codes.shape[1]
        self._hold(codes, scale)
        self._codes, self._scale = codes.data_ptr(), scale.data_ptr()

    def _made_of(self) -> tuple:
        return self.codes, self.scale, self.k


def pack_weight_i8(codes: torch.Tensor, scale: torch.Tensor) -> Int8Rows:
    """:class:`Int8Rows` from int8 ``codes`` [N, K] and fp32 ``scale`` [N] (a checkpoint's weight: one scale per output channel), laid out for
    :func:`gemm_i8` once."""
    if codes.dim() != 2 or codes.dtype != torch.int8 or not _on_gpu(codes) or not 1 <= codes.shape[1] <= _I8_MAX_K:
        raise ValueError(f"pack_weight_i8: codes must be a CUDA int8 [N, K] tensor, K <= {_I8_MAX_K}")
    if scale.dtype != torch.float32 or scale.shape != (codes.shape[0],) or scale.device != codes.device:
        raise ValueError(f"pack_weight_i8: scale must be fp32 [{codes.shape[0]}] on {codes.device}")
    if scale.requires_grad or forward_ad._current_level >= 0:
        _no_gradients("pack_weight_i8: scale", scale)
    n, k = codes.shape
    packed = torch.zeros((n, -(-k // 128) * 128), dtype=torch.int8, device=codes.device)
    packed[:, :k] = codes
    return Int8Rows(packed, scale.clone(memory_format=torch.contiguous_format), k)


_ONE_LAUNCH = 16384   # codes of up to 4 rows (half as many of up to 16) that mv_linear_i8 takes in one launch, without a workspace


def quantize_rows_i8(x: torch.Tensor) -> Int8Rows:
    """Each row of ``x`` [M, K] (fp16 | bf16) as int8 codes and one scale: scale = max|x| / 127, code = 127 x / max|x| rounded to nearest, ties
    to even.  A row of zeros has scale 0; a row that holds an infinity or NaN keeps that as its scale (its products are NaN)."""
    m, k, ld = _matrix(x, "x")
    if not 1 <= k <= _I8_MAX_K:
        raise ValueError(f"quantize_rows_i8: {k} columns (1 .. {_I8_MAX_K})")
    kp = -(-k // 128) * 128
    codes = torch.empty((m, kp), dtype=torch.int8, device=x.device)
    scale = torch.empty((m,), dtype=torch.float32, device=x.device)
    dev = x.get_device()
    with torch.cuda.device(dev):
        check(_lib.load().mv_quantize_rows_i8(x.data_ptr(), ld, m, k, _DTYPES[x.dtype], codes.data_ptr(), kp, scale.data_ptr(), _raw_stream(dev)),
              "mv_quantize_rows_i8")
    return Int8Rows(codes, scale, k)


def _i8_result(what: str, m: int, w: Int8Rows, like: torch.Tensor, dtype, bias, residual, act, out):
    """checks what the product is finished with; (bias, residual, out pointers, row strides of residual and out, out)"""
    dev, n = like.get_device(), w.rows
    if dtype not in _DTYPES:
        raise ValueError(f"{what}: dtype {dtype} (fp16, bf16)")
    if act not in (MV_ACT_NONE, MV_ACT_SILU):
        raise ValueError(f"{what}: activation {act}")
    if w._dev != dev:
        raise ValueError(f"{what}: weight on {w.device}, rows on {like.device}")
    if n < 1:
        raise ValueError(f"{what}: a weight without rows")
    if w.scale.requires_grad or forward_ad._current_level >= 0:
        _no_gradients(f"{what}: scale", w.scale)
    pb = pr = ldr = 0
    if bias is not None:
        pb = _affine(bias, f"{what}: bias", n, dtype, dev)
    if residual is not None:
        rows, cols, ldr = _matrix(residual, "residual", dtype, dev)
        if rows != m or cols != n:
            raise ValueError(f"{what}: residual {(rows, cols)}, the product is {(m, n)}")
        pr = residual.data_ptr()
    if out is None:
        out, ldo = torch.empty((m, n), dtype=dtype, device=like.device), n
    else:
        rows, cols, ldo = _matrix(out, "out", dtype, dev)
        if rows != m or cols != n:
            raise ValueError(f"{what}: out {(rows, cols)}, the product is {(m, n)}")
        _no_overlap(out, f"{what}: out", (("residual", residual), ("bias", bias)), ("residual",))
    return pb, pr, out.data_ptr(), ldr, ldo, out


def gemm_i8(a: Int8Rows, w: Int8Rows, *, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None, act: int = MV_ACT_NONE,
            dtype: torch.dtype = torch.float16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(a_scale[m] * w_scale[n] * sum_k a[m, k] w[n, k] + bias) + residual as ``dtype`` [M, N]; the sum of products is exact (int32).
    ``out`` may be ``residual`` itself."""
    if a.k != w.k:
        raise ValueError(f"gemm_i8: rows of {a.k}, weight of {w.k}")
    if a.scale.requires_grad or forward_ad._current_level >= 0:
        _no_gradients("gemm_i8: scale", a.scale)
    pb, pr, po, ldr, ldo, out = _i8_result("gemm_i8", a.rows, w, a.codes, dtype, bias, residual, act, out)
    _launch("mv_gemm_i8", _pack_gemm(a._codes, w._codes, a._scale, w._scale, pb, pr, po, a.rows, w.rows, w.kp, a.kp, w.kp, ldr, ldo, act, _DTYPES[dtype]),
            a._dev, (a, w))
    return out


def linear_i8(x: torch.Tensor, w: Int8Rows, *, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None, act: int = MV_ACT_NONE,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`gemm_i8` of :func:`quantize_rows_i8` (``x``) in one call: a projection whose weight and activations are multiplied in 8 bits."""
    m, k, ldx = _matrix(x, "x")
    dtype = x.dtype
    if k != w.k:
        raise ValueError(f"linear_i8: x {(m, k)}, weight of {w.k}")
    given = out is not None
    pb, pr, po, ldr, ldo, out = _i8_result("linear_i8", m, w, x, dtype, bias, residual, act, out)
    if given:
        _no_overlap(out, "linear_i8: out", (("x", x),))
    # mv_linear_i8's workspace: the rows' codes, then their scales; none where it quantises and multiplies in one launch
    ws = None if m <= 16 and m * w.kp <= (_ONE_LAUNCH if m <= 4 else _ONE_LAUNCH // 2) else torch.empty(m * (w.kp + 4), dtype=torch.uint8, device=x.device)
    _launch("mv_linear_i8", _pack_linear(x.data_ptr(), w._codes, w._scale, pb, pr, po, ws.data_ptr() if ws is not None else 0, m, w.rows, k, w.kp, ldx, w.kp, ldr, ldo, act,
                                         _DTYPES[dtype]), x.get_device(), (w,))
    return out
