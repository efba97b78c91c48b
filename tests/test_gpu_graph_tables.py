"""GPU tests: the table that a captured call reads lives as long as its graph, and no longer."""

import gc
import time

import pytest
import torch

from tests import packed_reference as R

pytestmark = pytest.mark.gpu


def rand(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16)


def settled(done):
    """Waits up to ten seconds: a graph lets go of what it held behind the back of the call that destroys it. What it let
    go of is freed by the next plan or call."""
    from b200_attention_b200 import ops

    for _ in range(200):
        ops.AttentionPlan([1], [1], heads=1)
        gc.collect()
        if done():
            return True
        time.sleep(0.05)
    return False


def captured(ops, plan, *inputs, calls=1):
    ops.attention_packed(*inputs, plan)  # the kernels are loaded
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [ops.attention_packed(*inputs, plan) for _ in range(calls)]
    return graph, out


def test_tables_go_with_their_graphs(native_built):
    from b200_attention_b200 import _native, ops

    n = 4000
    q, k, v = rand(1, n, 4, 128), rand(2, n, 2, 128), rand(3, n, 2, 128)
    before = []
    for _ in range(6):
        plan = ops.AttentionPlan([1] * n, [1] * n, heads=4, heads_kv=2)
        graph, out = captured(ops, plan, q, k, v, calls=3)
        graph.replay()
        torch.cuda.synchronize()
        table = plan._table.numel() * 4
        assert torch.equal(out[0], out[2])
        del graph, out, plan
        gc.collect()
        before.append(torch.cuda.memory_allocated())
    assert table > 500_000
    assert settled(lambda: torch.cuda.memory_allocated() < before[0] + table // 2)
    torch.cuda.synchronize()
    _native.device_check()


def test_a_table_stays_while_one_of_its_graphs_does(native_built):
    from b200_attention_b200 import _native, ops

    lens_q, lens_kv = [1, 40], [3000, 40]
    q, k, v = rand(1, 41, 8, 128), rand(2, 3040, 2, 128), rand(3, 3040, 2, 128)
    plan = ops.AttentionPlan(lens_q, lens_kv, heads=8, heads_kv=2)
    want = ops.attention_packed(q, k, v, plan)
    first, _ = captured(ops, plan, q, k, v)
    second, out = captured(ops, plan, q, k, v, calls=2)
    place, size = plan._table.data_ptr(), plan._table.numel()
    del plan, first
    for _ in range(10):
        ops.AttentionPlan([1], [1], heads=1)
        gc.collect()
        time.sleep(0.02)
    others = [torch.full((size,), -1, dtype=torch.int32, device="cuda") for _ in range(20)]
    assert place not in [t.data_ptr() for t in others]
    second.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in out)
    R.check_attention(want, None, R.attention(q, k, v, lens_q, lens_kv, causal=True))
    del out, others
    gc.collect()
    held = torch.cuda.memory_allocated()
    del second
    assert settled(lambda: torch.cuda.memory_allocated() <= held - 4 * size)
    _native.device_check()
