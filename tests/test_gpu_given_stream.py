"""GPU tests: what a call on a given stream reads may be let go of as soon as the call has returned."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def rand(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16)


def overwritten_behind(call, stream, make):
    """`call(*make())` on a stream that is busy, its inputs freed at once and their sizes allocated and filled anew."""
    torch.cuda.synchronize()
    tensors = make()
    for t in tensors:
        torch.zeros(1, dtype=t.dtype, device="cuda")  # the kernels that fill are loaded
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(400_000_000)
    got = call(*tensors)
    shapes = [(t.shape, t.dtype) for t in tensors]
    places = {t.data_ptr() for t in tensors}
    del tensors
    others = [torch.zeros(shape, dtype=dtype, device="cuda") for shape, dtype in shapes]
    assert not stream.query(), "the call was to be waiting still"
    assert not places & {t.data_ptr() for t in others}
    stream.synchronize()
    return got


def test_attention_on_a_given_stream(native_built):
    from b200_attention_b200 import _native, ops

    n, prefix = 700, 3000
    make = lambda: (rand(1, n, 8, 128), rand(2, prefix, 2, 128), rand(3, prefix, 2, 128), rand(4, n, 2, 128), rand(5, n, 2, 128))
    plan = ops.AttentionPlan([n], [n], heads=8, heads_kv=2)
    behind = ops.AttentionPlan([n], [n], heads=8, heads_kv=2, len_prefix=prefix)
    q, kp, vp, k, v = make()
    want = ops.attention_packed(q, k, v, plan), ops.attention_shared_prefix(q, kp, vp, k, v, behind)
    del q, kp, vp, k, v
    s = torch.cuda.Stream()
    got = overwritten_behind(lambda q, kp, vp, k, v: ops.attention_shared_prefix(q, kp, vp, k, v, behind, stream=s), s, make)
    assert torch.equal(got, want[1])
    got = overwritten_behind(lambda q, k, v: ops.attention_packed(q, k, v, plan, stream=s), s,
                             lambda: [t for i, t in enumerate(make()) if i in (0, 3, 4)])
    assert torch.equal(got, want[0])
    torch.cuda.synchronize()
    _native.device_check()


def test_rotation_on_a_given_stream(native_built):
    from b200_attention_b200 import _native, ops

    def make():
        return (rand(1, 900, 8, 128), rand(2, 900, 2, 128), torch.arange(900, device="cuda"),
                10000.0 ** (-torch.arange(64, device="cuda", dtype=torch.float32) / 64), rand(3, 128), rand(4, 128))

    s = torch.cuda.Stream()
    call = lambda q, k, pos, f, wq, wk, stream=s: ops.qk_norm_rope(q, k, pos, f, q_weight=wq, k_weight=wk, stream=stream)
    want = call(*make(), stream=None)
    got = overwritten_behind(call, s, make)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    torch.cuda.synchronize()
    _native.device_check()


def test_a_given_stream_that_is_being_captured(native_built):
    from b200_attention_b200 import _native, ops

    q, k, v = rand(1, 40, 8, 128), rand(2, 40, 2, 128), rand(3, 40, 2, 128)
    plan = ops.AttentionPlan([40], [40], heads=8, heads_kv=2)
    pos, f = torch.arange(40, device="cuda"), torch.ones(64, device="cuda")
    want, turned = ops.attention_packed(q, k, v, plan), ops.qk_norm_rope(q, k, pos, f)
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        s.wait_stream(torch.cuda.current_stream())
        got = ops.attention_packed(q, k, v, plan, stream=s)
        also = ops.qk_norm_rope(q, k, pos, f, stream=s)
        torch.cuda.current_stream().wait_stream(s)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(also[0], turned[0]) and torch.equal(also[1], turned[1])
    _native.device_check()
    del graph
