"""Attention over packed sequences of different lengths, and over requests that share a prefix.

    plan = AttentionPlan(lens_q, lens_kv, heads=32, heads_kv=8, causal=True)   # once per batch
    o = attention_packed(q, k, v, plan)                                        # every layer

    plan = AttentionPlan(lens_q, lens_kv, heads=32, heads_kv=8, len_prefix=len(k_prefix))
    o = attention_shared_prefix(q, k_prefix, v_prefix, k, v, plan)

Sequences lie back to back: q and o are [rows, heads, 128], k and v [rows, heads_kv, 128]; k and v may also be a
cache in which every sequence has rows of its own (`starts_kv`). A plan is made on the host from the lengths and
says which CTA works on what (see b200attn_plan_create); it depends on nothing else and serves every call with
those lengths. A whole prompt, a later chunk of one and a single new token are the same call with other lengths.

The reference project has no counterpart: its kernels take one rectangular problem.
"""

from __future__ import annotations

import ctypes as C
import operator
from typing import Optional

import torch

from . import _native as N


def _int_list(name: str, values) -> list:
    if isinstance(values, torch.Tensor):
        if values.is_cuda:
            raise RuntimeError(f"{name} must be host integers: a plan is made on the host")
        if values.dim() != 1 or values.dtype.is_floating_point or values.dtype in (torch.bool, torch.complex64):
            raise TypeError(f"{name} must be a 1-D tensor of integers")
        return values.tolist()
    out = []
    for v in values:
        i = v.__index__() if hasattr(v, "__index__") and not isinstance(v, bool) else None
        if i is None:
            raise TypeError(f"{name} must hold integers, got {v!r}")
        out.append(i)
    return out


class Schedule:
    """A plan's host side: sizes (`info`) and table (int32, host), from host arithmetic only."""

    def __init__(self, lens_q, lens_kv, *, heads: int, heads_kv: Optional[int] = None, causal: bool = True,
                 starts_kv=None, len_prefix: int = 0, sm_count: int = 0):
        lq, lk = _int_list("lens_q", lens_q), _int_list("lens_kv", lens_kv)
        if len(lq) != len(lk):
            raise ValueError(f"lens_q holds {len(lq)} lengths, lens_kv {len(lk)}")
        st = None if starts_kv is None else _int_list("starts_kv", starts_kv)
        if st is not None and len(st) != len(lk):
            raise ValueError(f"starts_kv holds {len(st)} rows, lens_kv {len(lk)} lengths")
        for name, vals, top in (("lens_q", lq, 2**30), ("lens_kv", lk, 2**30), ("starts_kv", st or (), 2**31)):
            if any(not 0 <= x < top for x in vals):
                raise ValueError(f"{name} must be 0 .. {top - 1}")
        heads, len_prefix = operator.index(heads), operator.index(len_prefix)
        heads_kv = heads if heads_kv is None else operator.index(heads_kv)
        for name, x in (("heads", heads), ("heads_kv", heads_kv), ("len_prefix", len_prefix)):
            if not -2**31 <= x < 2**31:
                raise ValueError(f"{name} is out of range")
        self.sequences, self.heads, self.heads_kv = len(lq), heads, heads_kv
        self.causal, self.len_prefix = bool(causal), len_prefix
        n = max(1, len(lq))
        d = N.PlanDesc()
        d.struct_bytes = C.sizeof(N.PlanDesc)
        d.sequences, d.heads, d.heads_kv = len(lq), self.heads, self.heads_kv
        d.causal, d.len_prefix, d.sm_count = int(self.causal), self.len_prefix, int(sm_count)
        d.len_q, d.len_kv = (C.c_int32 * n)(*lq), (C.c_int32 * n)(*lk)
        if st is not None:
            d.start_kv = (C.c_int64 * n)(*st)
        self.info = N.PlanInfo()
        self.info.struct_bytes = C.sizeof(N.PlanInfo)
        handle = C.c_void_p()
        lib = N.lib()
        N.check(lib.b200attn_plan_create(C.byref(d), C.byref(self.info), C.byref(handle)))
        try:
            self.table = torch.empty(self.info.table_bytes // 4, dtype=torch.int32)
            N.check(lib.b200attn_plan_table(handle, self.table.data_ptr(), self.info.table_bytes))
        finally:
            lib.b200attn_plan_destroy(handle)


class AttentionPlan:
    """Which CTA works on what, for sequences of the given lengths.

    lens_q, lens_kv: tokens and keys of each sequence (host integers; 0 allowed). heads_kv: K/V heads (default: as
    many as heads; query head h reads K/V head h // (heads // heads_kv)). causal: token i of n sees key j of m iff
    j <= i + (m - n), so a sequence's last token sees all of its keys. starts_kv: first row of each sequence in
    k and v; default: back to back. len_prefix: rows of a shared prefix that every token sees in front of its own
    keys (attention_shared_prefix). device: where the calls will run (default: the current CUDA device).

    `update` puts other lengths in place. Calls captured into a CUDA graph read the plan's table when the graph is
    replayed, so an updated plan changes what the replay does; `update` refuses lengths that a captured call has no
    room for. (What a replay does not compute, rows behind the new last sequence, keeps what the output held.) A plan
    may be used on any stream of its device, also by overlapping calls; only `update` must not overlap calls that use
    it on other streams than the current one. A graph keeps the table of its calls' plans for itself: it may be
    replayed after the plan is gone, and gives the table back when it is destroyed.
    """

    def __init__(self, lens_q, lens_kv, *, heads: int, heads_kv: Optional[int] = None, causal: bool = True,
                 starts_kv=None, len_prefix: int = 0, device=None):
        s = Schedule(lens_q, lens_kv, heads=heads, heads_kv=heads_kv, causal=causal, starts_kv=starts_kv,
                     len_prefix=len_prefix)
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise RuntimeError("a plan needs a CUDA device (this library has no CPU path)")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a plan cannot be made while the current stream is being captured")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        if torch.cuda.get_device_properties(device).multi_processor_count != 148:
            s = Schedule(lens_q, lens_kv, heads=heads, heads_kv=heads_kv, causal=causal, starts_kv=starts_kv,
                         len_prefix=len_prefix,
                         sm_count=min(160, torch.cuda.get_device_properties(device).multi_processor_count))
        self.device = device
        self.heads, self.heads_kv, self.causal, self.len_prefix = s.heads, s.heads_kv, s.causal, s.len_prefix
        self._sm_count = min(160, torch.cuda.get_device_properties(device).multi_processor_count)
        # room for the schedules of other lengths: twice this one's, and a little for small ones
        self._room_units = 2 * s.info.units + 1024
        self._room_slots = 2 * s.info.slot_rows + 4096
        self._captured = None  # (rows of q, rows of k) that every captured call has at least
        self._new_table(s)
        self._put(s)

    def _new_table(self, s: Schedule) -> None:
        N.direct().free_tables()
        self._table = torch.zeros(2 * s.table.numel() + 16384, dtype=torch.int32, device=self.device)
        self._table_stream = torch.cuda.current_stream(self.device).cuda_stream

    def _put(self, s: Schedule) -> None:
        with torch.cuda.device(self.device):
            # The copy is complete when this returns, so calls on any stream find the table. Host memory here is
            # pageable: nothing of it is read after that either.
            self._table[: s.table.numel()].copy_(s.table)
            torch.cuda.current_stream().synchronize()
        i = s.info
        self.rows_q, self.rows_kv = i.rows_q, i.rows_kv
        # what calls are told (serving_calls.h): sizes, launch, the launch of a captured call, for all that a later
        # table may hold, where the table was allocated, and which build of the kernel is the faster one
        self._now = (self.heads, self.heads_kv, i.rows_q, i.rows_kv, self.len_prefix, i.grid, i.units, i.slot_rows,
                     self._sm_count, self._room_units, self._room_slots, self._table_stream,
                     i.wide_pieces)

    def _hold(self, rows_q: int, rows_kv: int) -> None:
        held = self._captured or (rows_q, rows_kv)
        self._captured = (min(held[0], rows_q), min(held[1], rows_kv))

    def update(self, lens_q, lens_kv, *, starts_kv=None) -> None:
        """Other lengths, same heads, mask and prefix. Takes effect for calls made after it and for replays started
        after it, in the order of the current stream; waits for that stream."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a plan cannot be updated while the current stream is being captured")
        s = Schedule(lens_q, lens_kv, heads=self.heads, heads_kv=self.heads_kv, causal=self.causal,
                     starts_kv=starts_kv, len_prefix=self.len_prefix, sm_count=self._sm_count)
        fits = (s.table.numel() <= self._table.numel() and s.info.units <= self._room_units
                and s.info.slot_rows <= self._room_slots)
        if self._captured is not None:
            rows_q, rows_kv = self._captured
            if not fits or s.info.rows_q > rows_q or s.info.rows_kv > rows_kv:
                raise RuntimeError("these lengths do not fit the calls captured with this plan; make a new plan and "
                                   "capture again")
        elif not fits:
            self._room_units, self._room_slots = 2 * s.info.units + 1024, 2 * s.info.slot_rows + 4096
            self._new_table(s)
        self._put(s)


def used_on(stream: torch.cuda.Stream, *tensors) -> None:
    """What a call on a given stream reads or writes may be freed before it has run: its memory goes to nobody else until
    then. (A captured call's tensors are the caller's to keep, as with any captured call.)"""
    with torch.cuda.stream(stream):
        if torch.cuda.is_current_stream_capturing():
            return
    for t in tensors:
        if t is not None:
            t.record_stream(stream)


def _run(q, k, v, k_prefix, v_prefix, plan, softmax_scale, return_lse, out, stream):
    if stream is not None and stream != torch.cuda.current_stream(plan.device):
        if stream.device != plan.device:
            raise RuntimeError(f"stream is on {stream.device}, the plan on {plan.device}")
        with torch.cuda.stream(stream):
            result = _run(q, k, v, k_prefix, v_prefix, plan, softmax_scale, return_lse, out, None)
        used_on(stream, q, k, v, k_prefix, v_prefix, out)
        return result
    o, lse, captured = (N._direct or N.direct()).attention_planned(q, k, v, k_prefix, v_prefix, plan._table, plan._now,
                                                                   softmax_scale, return_lse, out)
    if captured:
        plan._hold(q.size(0), k.size(0))
    return (o, lse) if return_lse else o


def attention_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: AttentionPlan, *,
                     softmax_scale: float = 0.0, return_lse: bool = False, out: Optional[torch.Tensor] = None,
                     stream: Optional[torch.cuda.Stream] = None):
    """O = softmax(Q K^T * scale) V for every sequence of the plan, on the current CUDA stream.

    q: [rows, heads, 128] bf16, the sequences' tokens back to back; k, v: [rows, heads_kv, 128]. Any strides that are
    multiples of 8 elements (at least 128), head_dim dense. Returns O like q and, if asked, LSE [heads, rows] fp32
    (natural log). A token that sees no key gets O = 0 and LSE = -inf. Rows of q behind the plan's last sequence are
    not read; their rows of a given `out` keep what they hold, in an O made here they are 0 (LSE: -inf). Rows of
    k and v outside the plan's sequences have no influence, whatever they hold. `out` may be q itself, and otherwise
    must not overlap q, k, v or a prefix, nor itself. `stream`: where to launch instead of the current stream; what the
    call reads has to be there by that stream's order, and may be let go of once the call has returned.
    Forward only. softmax_scale <= 0: 1 / sqrt(128).
    """
    if not isinstance(plan, AttentionPlan):
        raise TypeError("plan must be an AttentionPlan")
    if plan.len_prefix:
        raise RuntimeError("this plan has a prefix: use attention_shared_prefix")
    return _run(q, k, v, None, None, plan, softmax_scale, return_lse, out, stream)


def attention_shared_prefix(q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor, k: torch.Tensor,
                            v: torch.Tensor, plan: AttentionPlan, *, softmax_scale: float = 0.0,
                            return_lse: bool = False, out: Optional[torch.Tensor] = None,
                            stream: Optional[torch.cuda.Stream] = None):
    """As attention_packed, with every token also seeing all of a prefix [len_prefix, heads_kv, 128] in front of its
    sequence's own keys. The prefix is read for blocks of tokens of all sequences together, not once per sequence.
    k_prefix, v_prefix: at least the plan's len_prefix rows (the first ones are used).
    """
    if not isinstance(plan, AttentionPlan):
        raise TypeError("plan must be an AttentionPlan")
    if not plan.len_prefix:
        raise RuntimeError("this plan has no prefix: use attention_packed")
    if k_prefix is None or v_prefix is None:
        raise TypeError("k_prefix and v_prefix must be torch.Tensors")
    return _run(q, k, v, k_prefix, v_prefix, plan, softmax_scale, return_lse, out, stream)


__all__ = ["AttentionPlan", "Schedule", "attention_packed", "attention_shared_prefix"]
