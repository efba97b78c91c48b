"""Norm of queries and keys for each head and their rotation by position, in one pass: what stands in front of an
attention call. The reference project has no counterpart (its model's own modules do this before they call it)."""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import _native as N
from .packed import used_on

def _same_place(a: torch.Tensor, b: torch.Tensor) -> bool:
    return N.direct().same_place(a, b)


def _may_overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    return N.direct().may_overlap(a, b)


def _dense_apart(t: torch.Tensor) -> bool:
    """True where no two elements of t share memory (expanded or overlapping windows do)."""
    return N.direct().dense_apart(t)


def _check_out(q, k, q_out, k_out) -> None:
    for name, t, needed in (("q", q, True), ("k", k, False)):
        if not isinstance(t, torch.Tensor) and (needed or t is not None):
            raise TypeError(f"{name} must be a torch.Tensor")
    pairs = [("q", q, q_out)] + ([("k", k, k_out)] if k is not None else [])
    for name, src, dst in pairs:
        if not isinstance(dst, torch.Tensor):
            raise TypeError(f"out of {name} must be a torch.Tensor")
        if dst.shape != src.shape or dst.dim() < 3:
            raise RuntimeError(f"out of {name} must match {name} in shape")
        if not _dense_apart(dst):
            raise RuntimeError(f"out of {name}: elements share memory")
    for name, _, dst in pairs:
        for other, src, _ in pairs:
            if not (name == other and _same_place(src, dst)) and _may_overlap(src, dst):
                raise RuntimeError(f"out of {name} overlaps {other} without being it")
    if k is not None and _may_overlap(q_out, k_out):
        raise RuntimeError("the outputs overlap")


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
    elements. `out`: tensors to write (q and k themselves, or apart from all inputs). One rounding to bf16, at the end. A
    value that is not finite reaches the other one of its pair, or with a norm all of its head, and no further.
    `stream`: where to launch instead of the current stream; what the call reads has to be there by that stream's order,
    and may be let go of once the call has returned.
    Forward only.
    """
    if sections is None:
        sections = (inv_freq.numel(),)
    elif type(sections) is not tuple:
        sections = tuple(sections)
    q_out = k_out = None
    if out is not None:
        q_out, k_out = out
        _check_out(q, k, q_out, k_out)
    if stream is not None and stream != torch.cuda.current_stream(q.device):
        if stream.device != q.device:
            raise RuntimeError(f"stream is on {stream.device}, q on {q.device}")
        with torch.cuda.stream(stream):
            result = _launch(q, k, positions, inv_freq, sections, q_weight, k_weight, eps, interleaved, q_out, k_out)
        used_on(stream, q, k, positions, inv_freq, q_weight, k_weight, q_out, k_out if k is not None else None)
        return result
    return _launch(q, k, positions, inv_freq, sections, q_weight, k_weight, eps, interleaved, q_out, k_out)


def _launch(q, k, positions, inv_freq, sections, q_weight, k_weight, eps, interleaved, q_out, k_out):
    done = (N._direct or N.direct()).qk_norm_rope(q, k, positions, inv_freq, sections, q_weight, k_weight, eps, interleaved,
                                                 q_out, k_out)
    if q_out is None:
        return done
    return q_out, k_out if k is not None else None


class QkNormRope:
    """qk_norm_rope with everything but q and k given once: what stands in front of a layer's attention. Accepted by
    backend.B200Attention, which applies it to query and key before it attends."""

    def __init__(self, positions: torch.Tensor, inv_freq: torch.Tensor, *, sections: Optional[Sequence[int]] = None,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 interleaved: bool = False):
        self.positions, self.inv_freq = positions, inv_freq
        self.options = dict(sections=None if sections is None else tuple(sections), q_weight=q_weight, k_weight=k_weight,
                            eps=eps, interleaved=interleaved)

    def __call__(self, q: torch.Tensor, k: Optional[torch.Tensor], *, out=None, stream=None):
        return qk_norm_rope(q, k, self.positions, self.inv_freq, out=out, stream=stream, **self.options)


__all__ = ["QkNormRope", "qk_norm_rope"]
