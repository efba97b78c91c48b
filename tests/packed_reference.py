"""Plain 64-bit forms of the packed / shared-prefix attention and of the norm-and-rotation, with error bounds.

Bounds of the attention kernels, element by element: every probability is rounded to bf16 once (relative 2^-8, the
row sum is taken before that rounding), so the weighted sum moves by at most 2^-8 * sum_j p_j |v_j|; the result is
rounded to bf16 once (2^-8 of its value). All else is in 32 bits: a product sum of 128 terms and the exponential of
a score (|score| < 30 in these tests) move a probability by less than 30 * 128 * 2^-24 < 2^-12 relative, and so the
weighted sum by less than 2^-11 of sum_j p_j |v_j| (numerator and row sum), which also covers the sums over up to
2^13 keys that the tensor cores and the row sums add up in 32 bits in blocks. LSE: the row sum's relative error,
2^-12, as an absolute one, and two roundings of a value below 2^5 in 32 bits.
"""

import math

import torch

HEAD_DIM = 128
HALF_STEP = 2.0 ** -8  # bf16


def starts_of(lens):
    out, at = [], 0
    for n in lens:
        out.append(at)
        at += n
    return out


def attention(q, k, v, lens_q, lens_kv, *, causal, starts=None, k_prefix=None, v_prefix=None, scale=None):
    """(O, LSE, sum_j p_j |v_j|), 64 bits, for the rows that the sequences cover."""
    starts = starts_of(lens_kv) if starts is None else starts
    heads, heads_kv = q.shape[1], k.shape[1]
    group = heads // heads_kv
    scale = HEAD_DIM ** -0.5 if scale is None else scale
    rows = sum(lens_q)
    o = torch.zeros(rows, heads, HEAD_DIM, dtype=torch.float64, device=q.device)
    spread = torch.zeros_like(o)
    lse = torch.full((heads, rows), -math.inf, dtype=torch.float64, device=q.device)
    at = 0
    for n, m, start in zip(lens_q, lens_kv, starts):
        ks, vs = k[start:start + m].double(), v[start:start + m].double()
        past = 0
        if k_prefix is not None:
            past = k_prefix.shape[0]
            ks, vs = torch.cat([k_prefix.double(), ks]), torch.cat([v_prefix.double(), vs])
        if n and past + m:
            ks, vs = (t.transpose(0, 1).repeat_interleave(group, 0) for t in (ks, vs))
            s = q[at:at + n].double().transpose(0, 1) @ ks.transpose(1, 2) * scale
            if causal:
                i = torch.arange(n, device=q.device)[:, None]
                j = torch.arange(past + m, device=q.device)[None]
                s = s.masked_fill(j > i + past + m - n, -math.inf)
            top = torch.logsumexp(s, -1, keepdim=True)
            p = torch.where(top == -math.inf, 0.0, torch.exp(s - top))
            o[at:at + n] = (p @ vs).transpose(0, 1)
            spread[at:at + n] = (p @ vs.abs()).transpose(0, 1)
            lse[:, at:at + n] = top[..., 0]
        at += n
    return o, lse, spread


def check_attention(o, lse, ref):
    o_ref, lse_ref, spread = ref
    rows = o_ref.shape[0]
    got = o[:rows].double()
    assert torch.isfinite(got).all()
    bound = (HALF_STEP + 2.0 ** -11) * spread + HALF_STEP * (o_ref.abs() + (HALF_STEP + 2.0 ** -11) * spread)
    worst = ((got - o_ref).abs() - bound).max().item() if rows else 0.0
    assert worst <= 0.0, f"an element is {worst:.3e} beyond its bound"
    if lse is not None:
        none = lse_ref == -math.inf
        assert torch.equal(lse[:, :rows] == -math.inf, none)
        off = (lse[:, :rows].double() - lse_ref)[~none].abs()
        assert off.numel() == 0 or off.max().item() <= 2.0 ** -12 + 2.0 ** -18


def rotate(x, weight, positions, inv_freq, sections, *, eps, interleaved):
    """64 bits; x [..., tokens, heads, 128], positions [axes, tokens] or [axes, batch, tokens]. Returns (y, bound)."""
    x = x.double()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    angle = (positions.double()[axis].movedim(0, -1) * inv_freq.double()).unsqueeze(-2)  # [.., tokens, 1, pairs]
    n = len(axis)
    first = torch.arange(n, device=x.device)
    a, b = (2 * first, 2 * first + 1) if interleaved else (first, first + HEAD_DIM // 2)
    y = x.clone()
    size = x.abs().clone()
    y[..., a] = x[..., a] * angle.cos() - x[..., b] * angle.sin()
    y[..., b] = x[..., b] * angle.cos() + x[..., a] * angle.sin()
    size[..., a] = size[..., b] = (x[..., a].square() + x[..., b].square()).sqrt()
    # One rounding to bf16. Before it, in 32 bits: the square sum (128 terms), its root and two products, relative
    # 2^-16 in all, and an angle off by 2 pi 2^-25, sine and cosine off by a few 2^-24, less than 2^-20: relative to
    # the pair's length.
    return y, HALF_STEP * y.abs() + 2.0 ** -15 * size
