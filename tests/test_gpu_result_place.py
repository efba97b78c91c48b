"""GPU tests: where the result of a packed or shared-prefix call may lie, and that other places are refused."""

import pytest
import torch

from tests import packed_reference as R

pytestmark = pytest.mark.gpu


def rand(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16)


def test_results_that_overlap_what_is_read_are_refused(native_built):
    from b200_attention_b200 import _native, ops

    rows = rand(1, 60, 4 + 2 + 2, 128)
    before = rows.clone()
    q, k, v = rows[:, :4], rows[:, 4:6], rows[:, 6:]
    plan = ops.AttentionPlan([40, 20], [40, 20], heads=4, heads_kv=2)
    behind = ops.AttentionPlan([40, 20], [40, 20], heads=4, heads_kv=2, len_prefix=30)
    prefix = rand(2, 120, 2, 128)
    twice = torch.zeros(61 * 512, device="cuda", dtype=torch.bfloat16)
    bad = [
        lambda: ops.attention_packed(q[:59], k, v, ops.AttentionPlan([59], [59], heads=4, heads_kv=2), out=rows[1:, :4]),
        lambda: ops.attention_packed(q, k, v, plan, out=rows[:, 1:5]),
        lambda: ops.attention_packed(q, k, v, plan, out=rows[:, 4:]),
        lambda: ops.attention_packed(q.contiguous(), k, v, plan, out=q.contiguous()[:, :1].expand(60, 4, 128)),
        lambda: ops.attention_packed(q.contiguous(), k, v, plan, out=twice.as_strided((60, 4, 128), (256, 128, 1))),
        lambda: ops.attention_shared_prefix(q, prefix[:60], prefix[60:], k, v, behind, out=prefix.view(60, 4, 128)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError, match="overlaps|share memory"):
            call()
            pytest.fail(f"call {i} was accepted")
    torch.cuda.synchronize()
    assert torch.equal(rows, before)
    _native.device_check()


def test_results_beside_the_inputs_or_in_the_place_of_q(native_built):
    """Columns of the same rows that nothing is read from, and q itself."""
    from b200_attention_b200 import _native, ops

    lens = [40, 1, 20]
    rows = rand(3, 61, 4 + 2 + 2 + 4, 128)
    q, k, v, beside = rows[:, :4], rows[:, 4:6], rows[:, 6:8], rows[:, 8:]
    plan = ops.AttentionPlan(lens, lens, heads=4, heads_kv=2)
    ref = R.attention(q, k, v, lens, lens, causal=True)
    for out in (beside, q):
        got = ops.attention_packed(q, k, v, plan, out=out)
        torch.cuda.synchronize()
        assert got is out or got.data_ptr() == out.data_ptr()
        R.check_attention(got, None, ref)
    _native.device_check()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_in_place_of_a_batch_with_heads_in_front_of_tokens(native_built, interleaved):
    from b200_attention_b200 import _native, ops

    buf = rand(5, 3, 4 + 2 + 2, 50, 128)                                   # [batch, heads of q, k and v, tokens, 128]
    q, k = buf[:, :4].transpose(1, 2), buf[:, 4:6].transpose(1, 2)
    pos = torch.arange(50, device="cuda")
    f = 10000.0 ** (-torch.arange(64, device="cuda", dtype=torch.float32) / 64)
    want_q, want_k = ops.qk_norm_rope(q, k, pos, f, interleaved=interleaved)
    v = buf[:, 6:].clone()
    ops.qk_norm_rope(q, k, pos, f, interleaved=interleaved, out=(q, k))
    torch.cuda.synchronize()
    assert torch.equal(q, want_q) and torch.equal(k, want_k) and torch.equal(buf[:, 6:], v)
    _native.device_check()


def test_rotated_rows_over_positions_frequencies_or_weights_are_refused(native_built):
    from b200_attention_b200 import _native, ops

    raw = torch.zeros(40 * 2 * 128 + 512, device="cuda", dtype=torch.bfloat16)
    out = raw[:40 * 2 * 128].view(40, 2, 128)
    before = raw.clone()
    pos, f, w = torch.arange(40, device="cuda"), torch.ones(64, device="cuda"), rand(2, 128)
    q = rand(1, 40, 2, 128)
    bad = [
        lambda: ops.qk_norm_rope(q, None, raw.view(torch.int64)[:40], f, out=(out, None)),
        lambda: ops.qk_norm_rope(q, None, pos, raw.view(torch.float32)[64:128], out=(out, None)),
        lambda: ops.qk_norm_rope(q, None, pos, f, q_weight=raw[256:384], out=(out, None)),
        lambda: ops.qk_norm_rope(rand(3, 40, 2, 128), q, pos, f, k_weight=raw[256:384], out=(torch.empty_like(q), out)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError, match="an output overlaps"):
            call()
            pytest.fail(f"call {i} was accepted")
    ops.qk_norm_rope(q, None, pos, raw[40 * 2 * 128:].view(torch.float32)[:64], q_weight=raw[-128:], out=(out, None))
    torch.cuda.synchronize()
    assert torch.equal(raw[40 * 2 * 128:], before[40 * 2 * 128:])
    _native.device_check()
