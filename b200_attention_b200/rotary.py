"""Norm of queries and keys for each head and their rotation by position, in one pass: what stands in front of an
attention call. The reference project has no counterpart (its model's own modules do this before they call it)."""

from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence, Tuple

import torch

from . import _native as N

HEAD_DIM = 128
_POSITION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}


def _check_tokens(name: str, t, like=None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (this library has no CPU path)")
    if t.dtype != torch.bfloat16:
        raise RuntimeError(f"{name} must be bfloat16, got {t.dtype}")
    if t.dim() not in (3, 4) or t.size(-1) != HEAD_DIM:
        raise RuntimeError(f"{name} must be [tokens, heads, {HEAD_DIM}] or [batch, tokens, heads, {HEAD_DIM}], "
                           f"got {tuple(t.shape)}")
    if t.stride(-1) != 1:
        raise RuntimeError(f"{name}: the head_dim axis must be contiguous")
    if like is not None:
        if t.device != like.device:
            raise RuntimeError(f"{name} is on {t.device}, q on {like.device}")
        if t.dim() != like.dim() or t.shape[:-2] != like.shape[:-2]:
            raise RuntimeError(f"{name} and q disagree on batch or tokens: {tuple(t.shape)}, {tuple(like.shape)}")


def _operand(t: torch.Tensor) -> N.Operand:
    # (batch, head, token); an axis of one entry is never stepped along
    stride = [0 if n == 1 else s for n, s in zip(t.shape, t.stride())]
    return N.Operand(t.data_ptr(), stride[0] if t.dim() == 4 else 0, stride[-2], stride[-3])


def _same_place(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and all(n == 1 or s == u for n, s, u in zip(a.shape, a.stride(), b.stride()))


def _span(t: torch.Tensor) -> Tuple[int, int]:
    first = t.data_ptr()
    return first, first + 2 * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _may_overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """False where two tensors cannot share an element: apart as a whole, or heads side by side in the same rows."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a1 <= b0 or b1 <= a0:
        return False
    if a.shape[:-2] == b.shape[:-2] and a.stride()[:-2] == b.stride()[:-2] and a.stride()[-2] == b.stride()[-2]:
        # the same rows, every row denser than the step to the next one: columns decide
        rows = [s for n, s in zip(a.shape[:-2], a.stride()[:-2]) if n > 1]
        width_a = 2 * ((a.size(-2) - 1) * a.stride(-2) + HEAD_DIM)
        width_b = 2 * ((b.size(-2) - 1) * b.stride(-2) + HEAD_DIM)
        reach = max(a0 + width_a, b0 + width_b) - min(a0, b0)
        nested = all(x >= 0 for x in rows) and (not rows or reach <= 2 * min(rows))
        if nested and (a0 + width_a <= b0 or b0 + width_b <= a0):
            return False
    return True


def _dense_apart(t: torch.Tensor) -> bool:
    """True where no two elements of t share memory (expanded or overlapping windows do)."""
    reach = 0
    for s, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if s <= reach:
            return False
        reach += s * (n - 1)
    return True


def qk_norm_rope(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    *,
    sections: Optional[Sequence[int]] = None,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    interleaved: bool = False,
    out: Optional[Tuple[torch.Tensor, Optional[torch.Tensor]]] = None,
    stream: Optional[torch.cuda.Stream] = None,
):
    """Returns (q', k'): every head of q and k normalised (where its weight is given) and turned by position.

    q: [tokens, heads, 128] or [batch, tokens, heads, 128] bf16; k: likewise with its own number of heads, or None.
    Per head: y = x * rsqrt(mean(x^2) + eps) * weight; then pair j of y, values (j, j + 64), or (2j, 2j + 1) if
    `interleaved`, is turned by positions[axis of j] * inv_freq[j]: (a, b) -> (a cos - b sin, b cos + a sin).
    sections: rotated pairs of each position axis (up to four axes, 64 pairs in all), in the order of the pairs:
    (16, 24, 24) turns pairs 0..15 by axis 0, 16..39 by axis 1, 40..63 by axis 2. Default: all of inv_freq by the
    only axis. Pairs behind the last section are not turned. inv_freq: [sum of sections] fp32.
    positions: int32, int64 or fp32, [axes, tokens], or [axes, batch, tokens]; [tokens] for one axis. Without a
    batch axis a batch's entries share them. Angles are worked out in 64 bits: far positions lose nothing.
    q_weight, k_weight: [128], both bf16 or both fp32, or None (no norm). Inputs need strides that are multiples of 8
    elements. `out`: tensors to write (may be q and k themselves). One rounding to bf16, at the end. Forward only.
    """
    _check_tokens("q", q)
    if k is not None:
        _check_tokens("k", k, q)
    elif k_weight is not None:
        raise RuntimeError("k_weight is given without k")
    batch, tokens = (q.size(0), q.size(1)) if q.dim() == 4 else (1, q.size(0))

    for name, t in (("positions", positions), ("inv_freq", inv_freq)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if t.device != q.device:
            raise RuntimeError(f"{name} is on {t.device}, q on {q.device}")
    if inv_freq.dim() != 1 or inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous():
        raise RuntimeError("inv_freq must be a contiguous fp32 vector")
    if positions.dtype not in _POSITION_TYPES:
        raise RuntimeError(f"positions must be int32, int64 or float32, got {positions.dtype}")
    sections = (inv_freq.numel(),) if sections is None else tuple(int(n) for n in sections)
    if not 1 <= len(sections) <= 4 or any(n < 0 for n in sections) or not 1 <= sum(sections) <= HEAD_DIM // 2:
        raise ValueError(f"sections must be 1 to 4 counts that add up to 1 .. {HEAD_DIM // 2}, got {sections}")
    if inv_freq.numel() != sum(sections):
        raise ValueError(f"inv_freq holds {inv_freq.numel()} frequencies, sections add up to {sum(sections)}")
    if positions.dim() == 1:
        positions = positions[None]
    if positions.dim() == 2 and tuple(positions.shape) == (len(sections), tokens):
        pos_batch = 0
    elif positions.dim() == 3 and tuple(positions.shape) == (len(sections), batch, tokens):
        pos_batch = positions.stride(1)
    else:
        raise RuntimeError(f"positions must be [{len(sections)}, {tokens}] or [{len(sections)}, {batch}, {tokens}], "
                           f"got {tuple(positions.shape)}")
    weights = [(n, w) for n, w in (("q_weight", q_weight), ("k_weight", k_weight)) if w is not None]
    for name, w in weights:
        if not isinstance(w, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if w.device != q.device or tuple(w.shape) != (HEAD_DIM,) or not w.is_contiguous() \
                or w.dtype not in (torch.bfloat16, torch.float32):
            raise RuntimeError(f"{name} must be a contiguous bf16 or fp32 vector of {HEAD_DIM} on q's device")
    if len({w.dtype for _, w in weights}) > 1:
        raise RuntimeError("q_weight and k_weight must have the same type")
    if torch.is_grad_enabled():
        for name, t in [("q", q), ("k", k), ("inv_freq", inv_freq), ("positions", positions)] + weights:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name} requires grad: this library computes forward passes only")
    if out is not None:
        q_out, k_out = out
        pairs = [("q", q, q_out)] + ([("k", k, k_out)] if k is not None else [])
        for name, src, dst in pairs:
            _check_tokens(f"out of {name}", dst, q)
            if dst.shape != src.shape:
                raise RuntimeError(f"out of {name} must match {name} in shape")
            if not _dense_apart(dst):
                raise RuntimeError(f"out of {name}: elements share memory")
        for name, _, dst in pairs:
            for other, src, _ in pairs:
                if not (name == other and _same_place(src, dst)) and _may_overlap(src, dst):
                    raise RuntimeError(f"out of {name} overlaps {other} without being it")
        if k is not None and _may_overlap(q_out, k_out):
            raise RuntimeError("the outputs overlap")

    def launch():
        s = torch.cuda.current_stream()
        if out is None:
            qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            ko = None if k is None else torch.empty(k.shape, dtype=k.dtype, device=k.device)
        else:
            qo, ko = out
            ko = None if k is None else ko
        if batch * tokens == 0 or q.size(-2) == 0:
            return qo, ko
        a = N.QkNormRopeArgs()
        a.struct_bytes = C.sizeof(N.QkNormRopeArgs)
        a.batch, a.tokens, a.heads_q, a.head_dim = batch, tokens, q.size(-2), HEAD_DIM
        a.q, a.q_out = _operand(q), _operand(qo)
        if k is not None and k.size(-2) > 0:
            a.heads_k, a.k, a.k_out = k.size(-2), _operand(k), _operand(ko)
        a.q_weight = q_weight.data_ptr() if q_weight is not None else None
        a.k_weight = k_weight.data_ptr() if k_weight is not None else None
        a.weight_type = int(bool(weights) and weights[0][1].dtype == torch.float32)
        a.position_type = _POSITION_TYPES[positions.dtype]
        a.positions = positions.data_ptr()
        a.position_stride_axis, a.position_stride_batch = positions.stride(0), pos_batch
        a.position_stride_token = positions.stride(-1)
        a.inv_freq = inv_freq.data_ptr()
        a.axes = len(sections)
        a.section[: len(sections)] = sections
        a.eps = float(eps)
        a.interleaved = int(bool(interleaved))
        a.stream = s.cuda_stream
        N.check(N.lib().b200attn_qk_norm_rope(C.byref(a)))
        return qo, ko

    if torch.cuda.current_device() != q.device.index:
        with torch.cuda.device(q.device):
            return _on(stream, launch)
    return _on(stream, launch)


def _on(stream, launch):
    if stream is not None and stream != torch.cuda.current_stream():
        with torch.cuda.stream(stream):
            return launch()
    return launch()


__all__ = ["qk_norm_rope"]
