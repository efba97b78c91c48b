"""Tensors that carry a tangent (forward-mode differentiation) are refused, as those that require a gradient are: these
calls compute neither."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from b200_attention_b200 import _native as N
from b200_attention_b200 import ops


def test_tangents_are_refused_before_a_device_is_touched(native_built):
    x, f, w = torch.zeros(4, 2, 128, dtype=torch.bfloat16), torch.zeros(64), torch.ones(128)
    pos = torch.arange(4)
    planned = lambda q, k, v: N.direct().attention_planned(q, k, v, None, None, torch.zeros(64, dtype=torch.int32),
                                                           (2, 2, 4, 4, 0, 1, 0, 0, 1, 0, 0, 0, 0), 0.0, False, None)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.qk_norm_rope(dual, x, pos, f), lambda: planned(dual, x, x)):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
    for call in (lambda: ops.qk_norm_rope(x, x, pos, f), lambda: planned(x, x, x)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


@pytest.mark.gpu
def test_tangents_are_refused(native_built):
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    q, k, v = (torch.randn(5, h, 128, generator=g, device="cuda", dtype=torch.bfloat16) for h in (4, 2, 2))
    pos = torch.arange(5, device="cuda")
    f, w = torch.rand(64, device="cuda"), torch.rand(128, device="cuda")
    plan = ops.AttentionPlan([5], [5], heads=4, heads_kv=2)
    shared = ops.AttentionPlan([5], [5], heads=4, heads_kv=2, len_prefix=2)
    want, rotated = ops.attention_packed(q, k, v, plan), ops.qk_norm_rope(q, k, pos, f, q_weight=w)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))
        bad = [
            lambda: ops.attention_packed(dual(q), k, v, plan),
            lambda: ops.attention_packed(q, dual(k), v, plan),
            lambda: ops.attention_packed(q, k, dual(v), plan),
            lambda: ops.attention_shared_prefix(q, dual(k), v, k, v, shared),
            lambda: ops.qk_norm_rope(dual(q), k, pos, f),
            lambda: ops.qk_norm_rope(q, dual(k), pos, f),
            lambda: ops.qk_norm_rope(q, k, dual(pos.float()), f),
            lambda: ops.qk_norm_rope(q, k, pos, dual(f)),
            lambda: ops.qk_norm_rope(q, k, pos, f, q_weight=dual(w)),
            lambda: ops.qk_norm_rope(q, k, pos, f, k_weight=dual(w)),
        ]
        for i, call in enumerate(bad):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
                pytest.fail(f"call {i} was accepted")
        # tensors without one are taken inside such a level
        assert torch.equal(ops.attention_packed(q, k, v, plan), want)
        assert torch.equal(ops.qk_norm_rope(q, k, pos, f, q_weight=w)[0], rotated[0])
    torch.cuda.synchronize()
    N.device_check()


@pytest.mark.gpu
def test_transforms_that_wrap_tensors_are_refused(native_built):
    """torch.func's transforms hand over wrappers without memory of their own."""
    q = torch.ones(5, 2, 128, device="cuda", dtype=torch.bfloat16)
    pos, f = torch.arange(5, device="cuda"), torch.rand(64, device="cuda")
    plan = ops.AttentionPlan([5], [5], heads=2)
    packed = lambda x: ops.attention_packed(x, q, q, plan)
    turned = lambda x: ops.qk_norm_rope(x, None, pos, f)[0]
    for call in (packed, turned):
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(q[None])
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (q,), (q,))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda x: call(x).float().sum())(q)
    torch.cuda.synchronize()
    N.device_check()
