"""What the probabilities' rounding does to rows with one dominating key, as trained models have on their first token."""

import pytest
import torch

from tests import packed_reference as R

pytestmark = pytest.mark.gpu


def sink_inputs(lens_q, lens_kv, heads, heads_kv, device="cuda"):
    """q, k, v in which the first key of every sequence has a score of 9 to 15 (another one for every row and head), the
    others about N(0, 1)."""
    g = torch.Generator(device=device)
    g.manual_seed(3)
    q, k, v = (torch.randn(n, h, R.HEAD_DIM, generator=g, device=device, dtype=torch.bfloat16)
               for n, h in ((sum(lens_q), heads), (sum(lens_kv), heads_kv), (sum(lens_kv), heads_kv)))
    q[..., 0] = 6 + 4 * torch.rand(q.shape[:2], generator=g, device=device)
    k[..., 0] = 0
    first = R.starts_of(lens_kv)
    k[first] = 0
    k[first, :, 0] = 17.0  # 17 * 6 / sqrt(128) = 9.0
    return q, k, v


def bound_of(q, k, v, lens_q, lens_kv):
    """(O, bound): as packed_reference's, but the largest probability of a row, its first key's, is 2^0 = 1 against the
    row's maximum and so is not rounded: only the others' share of sum_j p_j |v_j| moves by 2^-8 of itself."""
    o, lse, spread = R.attention(q, k, v, lens_q, lens_kv, causal=True)
    group = q.shape[1] // k.shape[1]
    largest = torch.empty_like(o)
    at = 0
    for n, start in zip(lens_q, R.starts_of(lens_kv)):
        k0, v0 = (t[start].double().repeat_interleave(group, 0) for t in (k, v))
        score = (q[at:at + n].double() * k0).sum(-1) * R.HEAD_DIM ** -0.5
        largest[at:at + n] = torch.exp(score - lse[:, at:at + n].T)[..., None] * v0.abs()
        at += n
    moved = R.HALF_STEP * (spread - largest) + 2.0 ** -11 * spread
    return o, moved + R.HALF_STEP * (o.abs() + moved)


@pytest.mark.parametrize("lens_q, lens_kv, heads, heads_kv", [
    ([1] * 40, [128] * 40, 8, 2),              # single tokens, one tile that every row sees all of
    ([1] * 24, [1024] * 24, 8, 2),
    ([1] * 3, [4096] * 3, 32, 8),              # cut into pieces
    ([128, 30], [256, 160], 4, 4),             # chunks behind a history, short
    ([1024], [1024], 4, 1),                    # prompts
    ([4096], [4096], 4, 2),
])
def test_a_dominating_key_is_not_rounded(native_built, lens_q, lens_kv, heads, heads_kv):
    from b200_attention_b200 import _native, ops

    q, k, v = sink_inputs(lens_q, lens_kv, heads, heads_kv)
    plan = ops.AttentionPlan(lens_q, lens_kv, heads=heads, heads_kv=heads_kv)
    got = ops.attention_packed(q, k, v, plan)
    torch.cuda.synchronize()
    _native.device_check()
    want, bound = bound_of(q, k, v, lens_q, lens_kv)
    beyond = ((got.double() - want).abs() - bound).max().item()
    assert beyond <= 0.0, f"an element is {beyond:.3e} beyond its bound"
